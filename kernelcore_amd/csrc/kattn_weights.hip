// kattn_weights.hip -- attn_weights_f16 / attn_weights_q4_0 (gfx950): what the query rows gave each cached position,
//   w_gj = decay w_in_gj + sum over rows r of KV head g of exp(y_rj - lse_r),
// with the scores y of flash_ext (kflash_ext_device.hpp). Tiles of 32 rows x 32 keys on the matrix cores, S = Q K^T (A = q rows, B =
// keys): lane (j, h) holds rows 8 (v / 4) + 4 h + v % 4 of key j, so a key's sum over the rows is a sum of registers and
// nothing crosses lanes until the end. A workgroup stages key tiles, and its wavefronts share the rows (RW of them
// to a tile). Sums in one order, no atomics.
// A single token's call reads K once. Over fp16 keys it is bound by that, or by a tile's latency (4099 positions, 8 KV heads of 128:
// 6.1 us); over 4-bit ones by unpacking them and multiplying tiles of 32 rows of which four are there (131072 positions: 38 us,
// 2 TB/s). With many rows the scaling of the sums and the exponentials bound it, and q, split anew for every 128 keys (64 tokens of 32 heads over
// 8192 4-bit positions: 19 us, 0.45 PFLOP/s counting both parts of q).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "internal.hpp"
#include "kflash_ext_device.hpp"

namespace kcamd {
namespace {

using namespace fx;

// What the rows gave a key whose sum came out NaN, from the definition, by a wavefront.
template <int D, bool Q4>
__device__ __forceinline__ void writePlainWeight(int kvh, int key, int lane) {
    const FxParams a = paramsAgain();
    float s = 0.0f;
    for (int r0 = 0; r0 < a.rows; r0 += 64) {
        const Row row = rowOf(a, kvh, r0 + lane);
        const float lse = a.lse[(size_t)row.token * a.H + row.head];
        if (row.live && lse != -INFINITY) s += expf(plainScore<D, Q4>(a, kvh, row, key) - lse);
    }
    s = waveSumF(s);
    const size_t at = (size_t)kvh * a.w_row + key;
    if (lane == 0) a.w[at] = a.w_in ? fmaf(a.decay, a.w_in[at], s) : s;
}

template <int D, bool Q4>
struct WGeo {
    static constexpr int NB = D / 32;
    static constexpr int oS = 32 * kKeyRow<D>, Tile = oS + (Q4 ? NB * 128 : 0);  // key rows, 4-bit: their blocks' scales
};

// RW wavefronts to a key tile, TP tiles to a wavefront: 4 / RW TP tiles to a workgroup of four (RW = 8: eight) wavefronts. Up to
// 64 rows (RW < 4) stay in registers, and the workgroup walks over the keys, the next ones' loads under way (131072 fp16
// positions of 8 heads of 128, one token: 45 us, 6 TB/s; a workgroup for every 128 keys, each with q of its own, 95); with more
// rows it walks over them, and has its keys only once. Two workgroups to a compute unit are worth some spilled registers at 256
// values (64 tokens over 8192: 34 against 47 us), but for a walk over fp16 keys (15 against 20).
// META: keys have positions or documents of their own, and tiles that no row sees are left out (a form of its own, whose registers
// cost the plain one 5%).
template <int RW>
constexpr int kWaves = RW > 4 ? RW : 4;
constexpr int kWalk = 256;  // the most steps of a walk
template <int D, bool Q4, int RW, int TP, bool META>
__global__ __launch_bounds__(64 * kWaves<RW>, D == 256 && RW == 1 && !Q4 ? 1 : 2) void attn_weights_kernel(FxParams a) {
    using G = WGeo<D, Q4>;
    constexpr int NB = G::NB, W = kWaves<RW>, NT = 64 * W, KW = W / RW, KT = KW * TP, PR = Q4 ? NB : D / 8, KS = D / 16;
    extern __shared__ int4 lds4[];
    __shared__ float part[W][TP][32];
    __shared__ float4 rows4[W][32];  // factor of the sums (base 2 unless capped), lse (base 2), slope, -
    __shared__ int4 rows4i[W][32];   // limit, position, document, token
    __shared__ unsigned long long lost[RW < 4 ? kWalk : 1][(KT + 1) / 2];  // a step's keys whose sums are NaN
    char* lds = reinterpret_cast<char*>(lds4);
    const int kvh = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31, h = lane >> 5;
    const int kw = wave / RW, rw = wave % RW;
    const char* kb = a.k + (size_t)kvh * a.k_head;
    const int* kpos = META && a.kpos ? a.kpos + (size_t)kvh * a.key_row : nullptr;
    const int* kdoc = META && a.kdoc ? a.kdoc + (size_t)kvh * a.key_row : nullptr;
    constexpr int IT = KT * 32 * PR, NL = (IT + NT - 1) / NT;
    u4 raw[NL];
    uint32_t sc[Q4 ? NL : 1];
    int rpos[TP], rdoc[TP];  // this lane's keys: key j of each of the wavefront's tiles
    auto load = [&](int t0) {
#pragma unroll
        for (int n = 0; n < NL; ++n) {
            const int i = tid + NT * n;
            if (i >= IT) break;
            const char* p = kb + (size_t)min((long long)t0 * 32 + i / PR, (long long)a.T - 1) * a.k_row + (Q4 ? 18 : 16) * (i % PR);
            if constexpr (Q4) {
                raw[n] = *reinterpret_cast<const u4a2*>(p + 2);
                sc[n] = loadHalf(p);
            } else {
                raw[n] = *reinterpret_cast<const u4a4*>(p);
            }
        }
#pragma unroll
        for (int p = 0; p < TP; ++p) {
            const int key = (int)min((long long)(t0 + kw * TP + p) * 32 + j, (long long)a.T - 1);
            rpos[p] = kpos ? kpos[key] : 0;
            rdoc[p] = kdoc ? kdoc[key] : 0;
        }
    };
    auto store = [&]() {
#pragma unroll
        for (int n = 0; n < NL; ++n) {
            const int i = tid + NT * n, key = i / PR, b = i % PR;
            if (i >= IT) break;
            char* tile = lds + (key >> 5) * G::Tile;
            if constexpr (Q4) {
                h8 code[4];
                blockCodes(raw[n], code);
                h8* dst = reinterpret_cast<h8*>(tile + (key & 31) * kKeyRow<D> + 64 * b);
#pragma unroll
                for (int e = 0; e < 4; ++e) dst[e] = code[e];
                reinterpret_cast<float*>(tile + G::oS)[b * 32 + (key & 31)] = finiteOrNaN(halfBits(sc[n]));
            } else {
                *reinterpret_cast<u4*>(tile + (key & 31) * kKeyRow<D> + 16 * b) = raw[n];
            }
        }
    };
    const Shape shape = shapeOf(a);
    f32x16 zero;
#pragma unroll
    for (int v = 0; v < 16; ++v) zero[v] = 0.0f;

    // a row tile: its rows' limits and documents; q as operands, what else its rows bring to LDS
    int r0 = 32 * rw, wmax = -1, wmin = INT_MAX, dmin = 0, dmax = 0;
    bool easy = false;  // whole, each of its rows saw something, and keys are hidden by position alone
    Row row;
    h8 qh[KS], ql[KS];
    auto limits = [&]() {
        row = rowOf(a, kvh, r0 + j);
        wmax = waveMax(row.live ? row.limit : -1);
        wmin = waveMin(row.live ? row.limit : INT_MAX);
        if (kdoc) {
            dmin = waveMin(row.doc);
            dmax = waveMax(row.doc);
        }
    };
    auto rows = [&]() {
        f32x4 q[D / 8];
        loadRow32<D>(a, row, h, q);
        const float lse = a.lse[(size_t)row.token * a.H + row.head];
        easy = !kpos && !kdoc && !a.mask && !__any(lse == -INFINITY) && r0 + 32 <= a.rows;
        const float c = splitRow32<D>(a, q, qh, ql);
        if (h == 0) {  // (a row that saw nothing gives nothing: its factor's place holds the mark)
            const bool none = !row.live || lse == -INFINITY;
            rows4[wave][j] = make_float4(shape.inv_cap > 0.0f ? c : factor2(c), none ? INFINITY : lse * kLog2e, row.slope, 0.0f);
            rows4i[wave][j] = make_int4(none ? -1 : row.limit, row.pos, row.doc, row.token);
        }
        waveLds();
    };
    const int tiles = a.T / 32 + (a.T % 32 != 0);
    int t0 = blockIdx.x * KT, step = 0;
    bool some = false;
    load(t0);
    if (RW < 4 && r0 < a.rows) {  // (the only one)
        limits();
        rows();
    }
    while (true) {
        const int key0 = (t0 + kw * TP) * 32, next = t0 + (int)gridDim.x * KT;
        const bool more = RW < 4 && next < tiles;
        store();
        int pos[TP], doc[TP];
#pragma unroll
        for (int p = 0; p < TP; ++p) {
            const long long key = (long long)key0 + 32 * p + j;
            pos[p] = key >= a.T ? kNoKey : kpos ? (rpos[p] < 0 ? kNoKey : rpos[p]) : (int)key;
            doc[p] = rdoc[p];
        }
        if (more) load(next);
        int first[TP], dlo[TP], dhi[TP];  // a tile's least position and its documents
#pragma unroll
        for (int p = 0; p < TP; ++p) {
            first[p] = kpos ? waveMin(pos[p]) : key0 + 32 * p;
            dlo[p] = kdoc ? waveMin(doc[p]) : 0;
            dhi[p] = kdoc ? waveMax(doc[p]) : 0;
        }
        auto seen = [&](int p) { return first[p] <= wmax && dlo[p] <= dmax && dhi[p] >= dmin; };  // by some row, perhaps
        __syncthreads();
        float acc[TP];
#pragma unroll
        for (int p = 0; p < TP; ++p) acc[p] = 0.0f;
        const auto products = [&]() {
            const int left = RW < 4 ? a.rows - r0 : 32;  // (groups of eight rows past the last one are left out)
#pragma unroll
            for (int p = 0; p < TP; ++p) {
                const int k0 = key0 + 32 * p;
                if (!seen(p)) continue;
                const char* tile = lds + (kw * TP + p) * G::Tile;
                const char* kr = tile + j * kKeyRow<D> + 16 * h;
                float x[16];
                if constexpr (Q4) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const h8 ka = *reinterpret_cast<const h8*>(kr + 64 * b), kc = *reinterpret_cast<const h8*>(kr + 64 * b + 32);
                        f32x16 s = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh[2 * b], ka, zero, 0, 0, 0);
                        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh[2 * b + 1], kc, s, 0, 0, 0);
                        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ql[2 * b], ka, s, 0, 0, 0);
                        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ql[2 * b + 1], kc, s, 0, 0, 0);
                        const float d = reinterpret_cast<const float*>(tile + G::oS)[b * 32 + j];
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            if (8 * g >= left) break;
#pragma unroll
                            for (int v = 4 * g; v < 4 * g + 4; ++v) x[v] = b ? fmaf(d, s[v], x[v]) : d * s[v];
                        }
                    }
                } else {
                    f32x16 s = zero;
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        const h8 ka = *reinterpret_cast<const h8*>(kr + 32 * k);
                        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh[k], ka, s, 0, 0, 0);
                        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ql[k], ka, s, 0, 0, 0);
                    }
#pragma unroll
                    for (int v = 0; v < 16; ++v) x[v] = s[v];
                }
                const bool full = easy && k0 + 31 <= wmin && k0 + 31 < a.T;
                if (full && shape.inv_cap == 0.0f && !shape.bias) {
#pragma unroll
                    for (int v = 0; v < 16; ++v) {
                        const float2 cl = *reinterpret_cast<const float2*>(&rows4[wave][8 * (v >> 2) + 4 * h + (v & 3)]);
                        acc[p] += ex2(fmaf(x[v], cl.x, -cl.y));
                    }
                    continue;
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {  // rows 8 g + 4 h .. + 4
                    if (8 * g >= left) break;
                    float y[4];
                    float4 rf[4];
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        rf[v] = rows4[wave][8 * g + 4 * h + v];
                        y[v] = x[4 * g + v] * rf[v].x;
                    }
                    if (shape.inv_cap > 0.0f) capScores<4>(y, shape.inv_cap, shape);
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        const int4 ri = rows4i[wave][8 * g + 4 * h + v];
                        if (shape.bias) y[v] = fmaf(-rf[v].z * kLog2e, fabsf((float)(ri.y - pos[p])), y[v]);
                        bool sees = pos[p] <= ri.x && doc[p] == ri.z;
                        if (a.mask && sees) {
                            const uint32_t mv = a.mask[(size_t)ri.w * a.m_row2 + k0 + j];
                            sees = mv != 0xFC00u;
                            y[v] = addMask(y[v], mv);
                        }
                        acc[p] += sees ? ex2(y[v] - rf[v].y) : 0.0f;
                    }
                }
            }
        };
        if constexpr (RW < 4) {
            if (r0 < a.rows) products();
        } else {
            for (r0 = 32 * rw; r0 < a.rows; r0 += 32 * RW) {
                limits();
                bool any = false;
#pragma unroll
                for (int p = 0; p < TP; ++p) any |= seen(p);
                if (!any) continue;
                rows();
                products();
                waveLds();
            }
        }
#pragma unroll
        for (int p = 0; p < TP; ++p) {
            acc[p] += __shfl_xor(acc[p], 32);
            if (h == 0) part[wave][p][j] = acc[p];
        }
        __syncthreads();
        if (wave < (KT + 1) / 2) {
            const int g = tid >> 5, w0 = g / TP * RW;
            const long long key = (long long)(t0 + g) * 32 + (tid & 31);
            const bool live = g < KT && key < a.T;
            float s = 0.0f;
            if (live) {
#pragma unroll
                for (int x = 0; x < RW; ++x) s += part[w0 + x][g % TP][tid & 31];
            }
            const unsigned long long nan = __ballot(s != s);
            if (lane == 0) lost[step][wave] = nan;
            some |= nan != 0;
            if (live && s == s) {
                const size_t at = (size_t)kvh * a.w_row + key;
                a.w[at] = a.w_in ? fmaf(a.decay, a.w_in[at], s) : s;
            }
        }
        ++step;
        if (!more) break;
        t0 = next;
    }
    if (__builtin_expect(some, 0)) {  // (each wavefront's own)
        for (int i = 0; i < step; ++i) {
            for (unsigned long long nan = lost[i][wave]; nan; nan &= nan - 1)
                writePlainWeight<D, Q4>(kvh, (int)((blockIdx.x + i * gridDim.x) * KT + 2 * wave) * 32 + __builtin_ctzll(nan), lane);
        }
    }
}

template <int D, bool Q4, int RW, int TP, bool META>
int runMeta(const FxParams& p, hipStream_t s) {
    constexpr int W = kWaves<RW>, kt = W / RW * TP, lds = WGeo<D, Q4>::Tile * kt;
    static const int ok = fromHip(hipFuncSetAttribute(reinterpret_cast<const void*>(attn_weights_kernel<D, Q4, RW, TP, META>),
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, lds), "attn_weights: LDS size");
    if (ok) return ok;
    const int tiles = p.T / 32 + (p.T % 32 != 0), all = (tiles + kt - 1) / kt;
    const int grid = RW < 4 ? std::min(all, std::max((all + kWalk - 1) / kWalk, (512 + p.H_kv - 1) / p.H_kv)) : all;  // (two workgroups to a compute unit)
    hipLaunchKernelGGL((attn_weights_kernel<D, Q4, RW, TP, META>), dim3(grid, p.H_kv), dim3(64 * W), lds, s, p);
    return fromHip(hipGetLastError(), "attn_weights");
}

template <int D, bool Q4, int RW, int TP>
int run(const FxParams& p, hipStream_t s) {
    return p.kpos || p.kdoc ? runMeta<D, Q4, RW, TP, true>(p, s) : runMeta<D, Q4, RW, TP, false>(p, s);
}

template <int D, bool Q4>
int runRows(const FxParams& p, hipStream_t s) {
    if (p.rows <= 32) return run<D, Q4, 1, 1>(p, s);
    if (p.rows <= 64) return run<D, Q4, 2, 1>(p, s);
    // four tiles to a wavefront, q read a quarter as often, where that leaves a workgroup for every compute unit; eight wavefronts
    // to a tile where there is no more than a tile for each (189 tokens over 759 positions, 24 heads of 128: 25 -> 16 us; 64 over
    // 2000, of 32: 12 -> 14)
    const long long keys = (long long)p.T * p.H_kv;
    if (keys >= 128 * 256) return run<D, Q4, 4, 4>(p, s);
    return p.rows > 128 && keys <= 32 * 256 ? run<D, Q4, 8, 1>(p, s) : run<D, Q4, 4, 1>(p, s);
}

}  // namespace

int launchAttnWeights(bool q4, const kcAttnWeightsArgs& a, hipStream_t s) {
    if (a.d.T == 0) return 0;
    FxParams p = fxParams(a.d, a.q, a.k, a.mask, a.qpos, a.kpos, a.qdoc, a.kdoc, a.slopes, a.scale, a.softcap);
    p.lse = const_cast<float*>(a.lse);
    p.w_in = a.w_in;
    p.w = a.w;
    p.w_row = a.w_row;
    p.decay = a.decay;
    switch (a.d.D) {
        case 64: return q4 ? runRows<64, true>(p, s) : runRows<64, false>(p, s);
        case 128: return q4 ? runRows<128, true>(p, s) : runRows<128, false>(p, s);
        case 256: return q4 ? runRows<256, true>(p, s) : runRows<256, false>(p, s);
        default: return fromHip(hipErrorInvalidValue, "attn_weights: D");
    }
}

}  // namespace kcamd
