// kflash_ext.hip -- flash_ext_f16 / flash_ext_q4_0 (gfx950): attention of N query tokens over T cached positions of an
// fp16 or a 4-bit cache with shaped scores: for query row i of a KV head (kflash_ext.hpp packs tokens and the
// group's heads into rows)
//   x_ij = cap tanh(scale q_i.k_j / cap) - slope_i |pos_i - pos_j| + mask_ij,   o_i = sum_j 2^(y_ij - m_i) v_j / l_i,
//   y = x log2 e, m_i = max_j y_ij, l_i = sum_j 2^(y_ij - m_i)
// over the keys that i sees, in one pass over the keys with running m and l.
//
// Three kernels: few rows (up to 32: single and drafted tokens), many rows (prompts), and the join of key ranges where
// a call's rows alone do not fill the GPU.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "internal.hpp"
#include "kflash_ext_device.hpp"

namespace kcamd {
namespace {

using namespace fx;

// p in [0, 1] is split into fp16 parts at this scale, so that what the parts cannot hold is below 2^-40
constexpr float kP = 32768.0f;

template <int N>
__device__ __forceinline__ float pick(const float* p, int i) {
    float r = p[0];
#pragma unroll
    for (int e = 1; e < N; ++e) r = i == e ? p[e] : r;
    return r;
}
// The value at dd of a V row that the matrix products left out (0 where they took it).
template <bool Q4>
__device__ float wildValue(const char* row, int dd) {
    if constexpr (Q4) {
        const char* b = row + 18 * (dd >> 5);
        const uint32_t s = loadHalf(b);
        if (!wildScale(s)) return 0.0f;
        const uint32_t c = (unsigned char)b[2 + (dd & 15)];
        return halfBits(s) * (float)((int)((dd & 16) ? c >> 4 : c & 15u) - 8);
    } else {
        const uint32_t x = loadHalf(row + 2 * dd);
        return (x & 0x7C00u) == 0x7C00u ? halfBits(x) : 0.0f;
    }
}

// ---------------------------------------------------------------------------------------------- many rows
// Workgroup: 128 rows of a KV head (four wavefronts of 32) over one range of keys, 32 keys at a time, which all four
// read from LDS; two buffers, the next keys' global loads in flight in registers while the present ones are
// computed. Matrix form (v_mfma_f32_32x32x16_f16, lane (j, h) = row j, lane half h):
//   S^T = K Q^T: A = key rows (LDS), B = q hi / lo (registers). Lane (j, h) holds keys 8 (v / 4) + 4 h + v % 4 of row j.
//   O^T += V^T P^T: A = V^T through transposed LDS reads, B = p hi / lo, the score registers as they are (the products'
//   index runs over the keys in the order those registers hold).
// 4-bit keys and values are unpacked once per workgroup, on the way to LDS.
template <int D, bool Q4>
struct Geo {
    static constexpr int NB = D / 32;
    static constexpr int KRow = kKeyRow<D>;
    static constexpr int VRow = 2 * D + 32;  // two, for the transposed reads
    static constexpr int oV = 32 * KRow, oVl = oV + 32 * VRow, oS = oV + 32 * VRow * (Q4 ? 2 : 1);
    static constexpr int oMeta = oS + (Q4 ? NB * 128 : 0);
    static constexpr int Buf = oMeta + 256;  // 32 positions, 32 document numbers
    static constexpr int MapWords = 1024;    // key tiles of a range, a bit each
    static constexpr int Lds = 2 * Buf + MapWords * 4 + 64;
};

template <int D, bool Q4, bool SHAPED>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void flash_ext_kernel(FxParams a) {
    using G = Geo<D, Q4>;
    constexpr int KS = D / 16, DB = D / 32, NB = G::NB;
    extern __shared__ int4 lds4[];
    char* lds = reinterpret_cast<char*>(lds4);
    uint32_t* map = reinterpret_cast<uint32_t*>(lds + 2 * G::Buf);
    int* misc = reinterpret_cast<int*>(map + G::MapWords);  // 0: largest limit, 1 / 2: least / largest document, 4 + i: wild keys
    const int kvh = blockIdx.x, rb = (int)gridDim.y - 1 - (int)blockIdx.y, sp = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31, h = lane >> 5;
    const Row row = rowOf(a, kvh, rb * 128 + wave * 32 + j);
    const int wmin = waveMin(row.live ? row.limit : INT_MAX), wmax = waveMax(row.live ? row.limit : -1);

    if (tid == 0) {
        misc[0] = -1;
        misc[1] = INT_MAX;
        misc[2] = INT_MIN;
    }
    if (tid >= 4 && tid < 8) misc[tid] = 0;
    __syncthreads();
    if (lane == 0) atomicMax(&misc[0], wmax);
    if (SHAPED && a.qdoc && row.live) {
        atomicMin(&misc[1], row.doc);
        atomicMax(&misc[2], row.doc);
    }
    __syncthreads();
    const int bmax = __builtin_amdgcn_readfirstlane(misc[0]);

    // this range's key tiles
    const bool meta = SHAPED && (a.kpos || a.kdoc);
    const int t0 = sp * a.per * 2;
    int t1 = (int)min((long long)t0 + 2LL * a.per, ((long long)a.T + 31) / 32);
    if (!(SHAPED && a.kpos)) t1 = bmax < 0 ? t0 : min(t1, bmax / 32 + 1);
    const int* kpos = SHAPED && a.kpos ? a.kpos + (size_t)kvh * a.key_row : nullptr;
    const int* kdoc = SHAPED && a.kdoc ? a.kdoc + (size_t)kvh * a.key_row : nullptr;
    const bool mapped = meta && t1 - t0 <= 32 * G::MapWords;
    if constexpr (SHAPED) {
        if (mapped) {  // the tiles that hold a position some row may see, in a document between the rows' least and largest
            const int dmin = misc[1], dmax = misc[2];
            for (int i = tid; i * 32 < t1 - t0; i += 256) map[i] = 0;
            __syncthreads();
            for (int t = t0 + 2 * wave; t < t1; t += 8) {
                const int key = t * 32 + lane;
                bool ok = key < a.T;
                if (ok && kpos) {
                    const int p = kpos[key];
                    ok = p >= 0 && p <= bmax;
                }
                if (ok && kdoc) {
                    const int x = kdoc[key];
                    ok = x >= dmin && x <= dmax;
                }
                const unsigned long long b = __ballot(ok);
                const uint32_t bits = ((uint32_t)b ? 1u : 0u) | ((uint32_t)(b >> 32) ? 2u : 0u);
                if (lane == 0 && bits) atomicOr(&map[(t - t0) >> 5], bits << ((t - t0) & 31));
            }
            __syncthreads();
        }
    }
    auto next = [&](int t) -> int {  // the first tile from t on that is to be computed; t1 if none
        if (!mapped) return min(t, t1);
        while (t < t1) {
            const uint32_t w = __builtin_amdgcn_readfirstlane(map[(t - t0) >> 5]) >> ((t - t0) & 31);
            if (w) return min(t + __builtin_ctz(w), t1);
            t = t0 + (((t - t0) >> 5) + 1) * 32;
        }
        return t1;
    };

    h8 qh[KS], ql[KS];
    const float c = loadRow32<D>(a, row, h, qh, ql);
    const Shape shape = shapeOf(a);
    const unsigned short* mrow = SHAPED && a.mask ? a.mask + (size_t)row.token * a.m_row2 : nullptr;

    // ---- staging: 16-byte chunks (fp16) or whole blocks (4-bit) of the tile's K and V rows, through registers
    constexpr int NL = Q4 ? (64 * NB + 255) / 256 : D / 32;  // chunks or blocks per thread
    u4 raw[NL];
    uint32_t rsc[Q4 ? NL : 1];
    int rmeta = 0;
    const char* kb = a.k + (size_t)kvh * a.k_head;
    const char* vb = a.v + (size_t)kvh * a.v_head;
    auto fetch = [&](int t) {
        if constexpr (Q4) {
#pragma unroll
            for (int n = 0; n < NL; ++n) {
                const int i = tid + 256 * n;
                if (i < 64 * NB) {
                    const bool isv = i >= 32 * NB;
                    const int ii = isv ? i - 32 * NB : i, key = t * 32 + ii / NB, b = ii % NB;
                    const size_t r = min(key, a.T - 1);
                    const char* p = (isv ? vb + r * a.v_row : kb + r * a.k_row) + 18 * b;
                    raw[n] = *reinterpret_cast<const u4a2*>(p + 2);
                    rsc[n] = isv && key >= a.T ? 0u : loadHalf(p);
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < NL; ++n) {  // the first half of the chunks K, the second V
                const bool isv = n >= NL / 2;
                const int i = tid + 256 * (isv ? n - NL / 2 : n), key = t * 32 + i / (D / 8), ch = i % (D / 8);
                const size_t r = min(key, a.T - 1);
                raw[n] = *reinterpret_cast<const u4a4*>((isv ? vb + r * a.v_row : kb + r * a.k_row) + 16 * ch);
                if (isv && key >= a.T) raw[n] = u4{0, 0, 0, 0};
            }
        }
        if constexpr (SHAPED) {
            if (meta && tid < 64) {
                const int key = t * 32 + (tid & 31);
                if (tid < 32) {
                    const int p = key < a.T ? (kpos ? kpos[key] : key) : kNoKey;
                    rmeta = p < 0 ? kNoKey : p;
                } else {
                    rmeta = kdoc && key < a.T ? kdoc[key] : 0;
                }
            }
        }
    };
    auto store = [&](char* buf, int* wild) {
        if constexpr (Q4) {
#pragma unroll
            for (int n = 0; n < NL; ++n) {
                const int i = tid + 256 * n;
                if (i < 64 * NB) {
                    const bool isv = i >= 32 * NB;
                    const int ii = isv ? i - 32 * NB : i, key = ii / NB, b = ii % NB;
                    h8 code[4];
                    blockCodes(raw[n], code);
                    if (!isv) {
                        h8* p = reinterpret_cast<h8*>(buf + key * G::KRow + 64 * b);
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[e] = code[e];
                        reinterpret_cast<float*>(buf + G::oS)[b * 32 + key] = halfBits(rsc[n]);
                    } else {
                        uint32_t s = rsc[n];
                        if (wildScale(s)) {
                            s = 0;
                            atomicOr(wild, 1 << key);
                        }
                        const _Float16 d = __builtin_bit_cast(_Float16, (unsigned short)s);
                        const _Float16 dh = __builtin_bit_cast(_Float16, (unsigned short)(s & 0xFFF0u));
                        const _Float16 dl = d - dh;
                        h8* p = reinterpret_cast<h8*>(buf + G::oV + key * G::VRow + 64 * b);
                        h8* pl = reinterpret_cast<h8*>(buf + G::oVl + key * G::VRow + 64 * b);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            p[e] = code[e] * dh;
                            pl[e] = code[e] * dl;
                        }
                    }
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < NL; ++n) {
                const bool isv = n >= NL / 2;
                const int i = tid + 256 * (isv ? n - NL / 2 : n), key = i / (D / 8), ch = i % (D / 8);
                u4 x = raw[n];
                if (isv) {
                    const uint32_t any = wildHalves(x[0]) | wildHalves(x[1]) | wildHalves(x[2]) | wildHalves(x[3]);
                    if (any) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t z = wildHalves(x[w]);
                            x[w] &= ~((z >> 15 & 1u) * 0xFFFFu | (z >> 31) * 0xFFFF0000u);
                        }
                        atomicOr(wild, 1 << key);
                    }
                }
                *reinterpret_cast<u4*>(buf + (isv ? G::oV + key * G::VRow : key * G::KRow) + 16 * ch) = x;
            }
        }
        if constexpr (SHAPED)
            if (meta && tid < 64) reinterpret_cast<int*>(buf + G::oMeta)[tid] = rmeta;
    };

    f32x16 zero;
#pragma unroll
    for (int v = 0; v < 16; ++v) zero[v] = 0.0f;
    f32x16 o[DB];
#pragma unroll
    for (int t = 0; t < DB; ++t) o[t] = zero;
    float m = -INFINITY, l = 0.0f;

    int t = next(t0);
    int slot = 0;  // of the wild-key words: three in turn, the one two tiles on is cleared while none reads it
    if (t < t1) {
        fetch(t);
        store(lds, &misc[4]);
    }
    __syncthreads();
    const int vlane = (4 * (lane >> 5) + ((lane & 15) >> 2)) * (G::VRow / 2) + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    for (int it = 0; t < t1; ++it) {
        const int tn = next(t + 1);
        char* cur = lds + (it & 1) * G::Buf;
        if (tn < t1) fetch(tn);
        const bool full = !meta && !(SHAPED && mrow) && t * 32 + 31 <= wmin && t * 32 + 31 < a.T;
        if (full || meta || t * 32 <= wmax) {
            MaskWords mk;
            if constexpr (SHAPED) {
                if (mrow) mk.load(mrow, t, h, a.T);
            }
            float x[16];
            keyScores<D, Q4>(cur, cur + G::oS, j, h, qh, ql, x);
            if constexpr (SHAPED) {
                shapeScores(x, c, shape, row, meta ? reinterpret_cast<const int*>(cur + G::oMeta) : nullptr, mrow ? &mk : nullptr, t, h);
            } else {
                const float c2 = c * kLog2e;
#pragma unroll
                for (int v = 0; v < 16; ++v) x[v] *= c2;
            }
            if (!meta && !full) {
                const int last = min(row.limit, a.T - 1) - t * 32 - 4 * h;
#pragma unroll
                for (int v = 0; v < 16; ++v) x[v] = 8 * (v >> 2) + (v & 3) <= last ? x[v] : -INFINITY;
            }
            float bm = x[0];
#pragma unroll
            for (int v = 1; v < 16; ++v) bm = fmaxf(bm, x[v]);
            bm = fmaxf(bm, __shfl_xor(bm, 32));
            const float mn = fmaxf(m, bm);
            const float ms = mn == -INFINITY ? 0.0f : mn;  // (nothing seen yet: every p is 0)
            if (__any(mn > m)) {
                const float alpha = ex2(m - ms);
                l *= alpha;
#pragma unroll
                for (int t2 = 0; t2 < DB; ++t2)
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[t2][v] *= alpha;
                m = mn;
            }
            h8 ph[2], pl[2];
            float ls = 0.0f;
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                x[v] = ex2(x[v] - ms);
                ls += x[v];
            }
            l += ls;
            uint32_t wild = __builtin_amdgcn_readfirstlane(misc[4 + slot]);
            while (__builtin_expect(wild != 0, 0)) {  // values that are no matrix operands, for the rows that see them
                const int key = __builtin_ctz(wild);
                wild &= wild - 1;
                const float p = __shfl(pick<16>(x, (key >> 3) * 4 + (key & 3)), j + 32 * ((key >> 2) & 1)) * kP;
                const char* vr = vb + (size_t)(t * 32 + key) * a.v_row;
#pragma unroll
                for (int t2 = 0; t2 < DB; ++t2)
#pragma unroll
                    for (int v = 0; v < 16; ++v) {
                        const float z = wildValue<Q4>(vr, 32 * t2 + 8 * (v >> 2) + 4 * h + (v & 3));
                        if (p != 0.0f && z != 0.0f) o[t2][v] = fmaf(p, z, o[t2][v]);
                    }
            }
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                const float ps = x[v] * kP;
                const _Float16 hi = (_Float16)ps;
                ph[v >> 3][v & 7] = hi;
                pl[v >> 3][v & 7] = (_Float16)(ps - (float)hi);
            }
            const _Float16* vcol = reinterpret_cast<const _Float16*>(cur + G::oV) + vlane;
#pragma unroll
            for (int mm = 0; mm < 2; ++mm)
#pragma unroll
                for (int t2 = 0; t2 < DB; ++t2) {
                    const _Float16* vp = vcol + 16 * mm * (G::VRow / 2) + 32 * t2;
                    const s4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)vp);
                    const s4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(vp + 8 * (G::VRow / 2)));
                    const h8 va = __builtin_bit_cast(h8, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
                    o[t2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, ph[mm], o[t2], 0, 0, 0);
                    o[t2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl[mm], o[t2], 0, 0, 0);
                    if constexpr (Q4) {
                        const _Float16* vq = vp + (G::oVl - G::oV) / 2;
                        const s4 y0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)vq);
                        const s4 y1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(vq + 8 * (G::VRow / 2)));
                        const h8 vl = __builtin_bit_cast(h8, __builtin_shufflevector(y0, y1, 0, 1, 2, 3, 4, 5, 6, 7));
                        o[t2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph[mm], o[t2], 0, 0, 0);
                    }
                }
        }
        // the next tile into the other buffer (read last two tiles ago, before the barrier below)
        const int sn = slot == 2 ? 0 : slot + 1, sc = sn == 2 ? 0 : sn + 1;
        if (tn < t1) store(lds + ((it + 1) & 1) * G::Buf, &misc[4 + sn]);
        if (tid == 0) misc[4 + sc] = 0;
        slot = sn;
        t = tn;
        __syncthreads();
    }

    l += __shfl_xor(l, 32);
    if (!row.live) return;
    const int r = rb * 128 + wave * 32 + j;
    float* dst;
    float f;
    if (a.splits == 1) {
        dst = a.out + ((size_t)row.token * a.H + row.head) * D;
        f = l == 0.0f ? 0.0f : 1.0f / (l * kP);
        if (a.lse && h == 0) a.lse[(size_t)row.token * a.H + row.head] = l == 0.0f ? -INFINITY : fmaf(m, kLn2, logf(l));
    } else {
        dst = a.part + (((size_t)sp * a.H_kv + kvh) * a.rows + r) * (D + 2);
        f = 1.0f / kP;
        if (h == 0) {
            dst[D] = m;
            dst[D + 1] = l;
        }
    }
#pragma unroll
    for (int t2 = 0; t2 < DB; ++t2)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 y = {o[t2][4 * g] * f, o[t2][4 * g + 1] * f, o[t2][4 * g + 2] * f, o[t2][4 * g + 3] * f};
            *reinterpret_cast<f4a4*>(dst + 32 * t2 + 8 * g + 4 * h) = y;
        }
}

// ---------------------------------------------------------------------------------------------- few rows
// Up to 32 rows (NR columns of 16): single tokens and a few drafted ones, where the cache's bytes count. Workgroup: four
// wavefronts over one range of keys of a KV head, each with its own tiles (64 keys of a 4-bit cache, 32 of an fp16
// one), joined through LDS at the end. v_mfma_f32_16x16x32_f16, lane (i, kg) = column i, group kg of 16 lanes:
//   S^T = K Q^T: fp16 keys are loaded as the A operand straight from memory; 4-bit keys go through LDS as they are, lane (i, kg)
//   unpacks word kg of a block of key i, the 32 values of a block are one step of the products, and its scale multiplies the
//   step's f32 sums. Lane (i, kg) then holds keys 16 u + 4 kg + v of row i.
//   O^T += V^T P^T: 4-bit values are transposed as they are (ds_read_b64_tr_b4: 16 keys of one value per lane), then unpacked
//   and scaled; fp16 values through 16-bit transposed reads.
template <int D, bool Q4, int NR>
struct FewGeo {
    static constexpr int NB = D / 32, TK = Q4 ? 64 : 32;
    static constexpr int Row = D / 2 + 16;   // LDS bytes of a key's codes
    static constexpr int VRow = 2 * D + 32;  // of an fp16 row
    static constexpr int oV = 64 * Row, oS = 2 * oV, oD = oS + NB * 256;  // 4-bit: codes of K, of V, K scales, V scales
    static constexpr int Wave = Q4 ? oD + NB * 256 : 32 * VRow;
    static constexpr int ORow = D + 4;       // join: floats per row
    static constexpr int Join = 4 * NR * 16 * (ORow + 2) * 4;
    static constexpr int Lds = 4 * Wave > Join ? 4 * Wave : Join;
};

// The lanes' loads and stores of LDS before this are done before those after it (a wavefront's own LDS accesses run in
// order: only the compiler has to keep them so).
__device__ __forceinline__ void waveLds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <int D, bool Q4, bool SHAPED, int NR>
__global__ __launch_bounds__(256, D == 256 || NR == 2 ? 1 : 2) void flash_ext_few_kernel(FxParams a) {
    using G = FewGeo<D, Q4, NR>;
    constexpr int NB = G::NB, TK = G::TK, U = TK / 16, TT = TK / 32, DT = D / 16;
    extern __shared__ int4 lds4[];
    char* lds = reinterpret_cast<char*>(lds4);
    const int sp = blockIdx.x, kvh = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i = lane & 15, kg = lane >> 4;
    char* mine = lds + wave * G::Wave;
    Row row[NR];
    int wmin = INT_MAX, wmax = -1;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        row[n] = rowOf(a, kvh, 16 * n + i);
        if (row[n].live) {
            wmin = min(wmin, row[n].limit);
            wmax = max(wmax, row[n].limit);
        }
    }
    wmin = waveMin(wmin);
    wmax = waveMax(wmax);
    const bool meta = SHAPED && (a.kpos || a.kdoc);
    const int* kpos = SHAPED && a.kpos ? a.kpos + (size_t)kvh * a.key_row : nullptr;
    const int* kdoc = SHAPED && a.kdoc ? a.kdoc + (size_t)kvh * a.key_row : nullptr;
    const int t0 = sp * a.per * (64 / TK);
    int t1 = (int)min((long long)t0 + (long long)a.per * (64 / TK), ((long long)a.T + TK - 1) / TK);
    if (!kpos) t1 = wmax < 0 ? t0 : min(t1, wmax / TK + 1);

    // q as the B operand of step b (32 values): fp16 keys: values 32 b + 8 kg + e; 4-bit keys: the order nibbles() gives
    h8 qh[NR][NB], ql[NR][NB];
    float c[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const float* qp = a.q + (size_t)row[n].token * a.q_tok + (size_t)row[n].head * a.q_head + (Q4 ? 4 : 8) * kg;
        float x[NB][8], top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const f32x4 u = *reinterpret_cast<const f4a4*>(qp + 32 * b), w = *reinterpret_cast<const f4a4*>(qp + 32 * b + (Q4 ? 16 : 4));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int nib = (e >> 1) + 4 * (e & 1);
                x[b][e] = Q4 ? (nib & 1 ? w[nib >> 1] : u[nib >> 1]) : (e < 4 ? u[e & 3] : w[e & 3]);
                top = fmaxf(top, fabsf(x[b][e]));
            }
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const QScale qs = qScale(top, a.scale);
        c[n] = qs.c;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                _Float16 hi, lo;
                qSplit(x[b][e], a.scale < 0.0f, qs.shift, hi, lo);
                qh[n][b][e] = hi;
                ql[n][b][e] = lo;
            }
    }
    const Shape shape = shapeOf(a);
    const char* kb = a.k + (size_t)kvh * a.k_head;
    const char* vb = a.v + (size_t)kvh * a.v_head;

    // a tile's loads. 4-bit: blocks lane + 64 n of the tile's 64 NB. fp16: K as the A operand [u][b], V chunks lane + 64 n.
    u4 kr[Q4 ? NB : 2 * NB], vr[Q4 ? NB : 2 * NB];
    uint32_t ks[Q4 ? NB : 1], vs[Q4 ? NB : 1];
    auto fetch = [&](int t) {
        if constexpr (Q4) {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const int ii = lane + 64 * n, key = t * 64 + ii / NB, b = ii % NB;
                const size_t r = min(key, a.T - 1);
                const char *kp = kb + r * a.k_row + 18 * b, *vp = vb + r * a.v_row + 18 * b;
                kr[n] = *reinterpret_cast<const u4a2*>(kp + 2);
                ks[n] = loadHalf(kp);
                vr[n] = *reinterpret_cast<const u4a2*>(vp + 2);
                vs[n] = key < a.T ? loadHalf(vp) : 0u;
            }
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const size_t r = min(t * 32 + 16 * u + i, a.T - 1);
#pragma unroll
                for (int b = 0; b < NB; ++b)
                    kr[u * NB + b] = *reinterpret_cast<const u4a4*>(kb + r * a.k_row + 64 * b + 16 * kg);
            }
#pragma unroll
            for (int n = 0; n < 2 * NB; ++n) {
                const int ii = lane + 64 * n, key = t * 32 + ii / (D / 8), ch = ii % (D / 8);
                const size_t r = min(key, a.T - 1);
                vr[n] = *reinterpret_cast<const u4a4*>(vb + r * a.v_row + 16 * ch);
                if (key >= a.T) vr[n] = u4{0, 0, 0, 0};
            }
        }
    };

    f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 o[NR][DT];
    float m[NR], l[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
        for (int t = 0; t < DT; ++t) o[n][t] = zero;
        m[n] = -INFINITY;
        l[n] = 0.0f;
    }
    // the key whose codes this lane addresses in the transposed reads: nibble x of word w of a lane's result is element
    // 2 (x % 4) + x / 4 of tile half w, and element e is key 32 w + 16 (e / 4) + 4 kg + e % 4
    const int xn = i & 7, en = 2 * (xn & 3) + (xn >> 2);
    const int trow = 32 * (i >> 3) + 16 * (en >> 2) + 4 * kg + (en & 3);

    int t = t0 + wave;
    if (t < t1) fetch(t);
    for (; t < t1; t += 4) {
        bool wild = false;
        h8 ka[Q4 ? 1 : 2 * NB];
        if constexpr (Q4) {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const int ii = lane + 64 * n, key = ii / NB, b = ii % NB;
                *reinterpret_cast<u4*>(mine + key * G::Row + 16 * b) = kr[n];
                *reinterpret_cast<u4*>(mine + G::oV + key * G::Row + 16 * b) = vr[n];
                reinterpret_cast<float*>(mine + G::oS)[b * 64 + key] = halfBits(ks[n]);
                uint32_t s = vs[n];
                if (wildScale(s)) {
                    s = 0;
                    wild = true;
                }
                const uint32_t dh = s & 0xFFF0u;
                const _Float16 dl = __builtin_bit_cast(_Float16, (unsigned short)s) - __builtin_bit_cast(_Float16, (unsigned short)dh);
                // in the order of the products: [block][tile half][kg][16-key half, key % 4]
                const int at = ((b * 2 + (key >> 5)) * 4 + ((key & 15) >> 2)) * 8 + 4 * ((key >> 4) & 1) + (key & 3);
                unsigned short* vd = reinterpret_cast<unsigned short*>(mine + G::oD);
                vd[at] = (unsigned short)dh;
                vd[64 * NB + at] = __builtin_bit_cast(unsigned short, dl);
            }
        } else {
#pragma unroll
            for (int n = 0; n < 2 * NB; ++n) {
                const int ii = lane + 64 * n, key = ii / (D / 8), ch = ii % (D / 8);
                u4 x = vr[n];
                const uint32_t any = wildHalves(x[0]) | wildHalves(x[1]) | wildHalves(x[2]) | wildHalves(x[3]);
                if (any) {
                    wild = true;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t z = wildHalves(x[w]);
                        x[w] &= ~((z >> 15 & 1u) * 0xFFFFu | (z >> 31) * 0xFFFF0000u);
                    }
                }
                *reinterpret_cast<u4*>(mine + key * G::VRow + 16 * ch) = x;
                ka[n] = __builtin_bit_cast(h8, kr[n]);
            }
        }
        const bool more = t + 4 < t1;
        if (more) fetch(t + 4);
        waveLds();
        float x[NR][U * 4];
        if constexpr (Q4) {
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int v = 0; v < U * 4; ++v) x[n][v] = 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const h8 kk = nibbles(*reinterpret_cast<const uint32_t*>(mine + (16 * u + i) * G::Row + 16 * b + 4 * kg));
                    const f32x4 d = *reinterpret_cast<const f32x4*>(mine + G::oS + (b * 64 + 16 * u + 4 * kg) * 4);
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        f32x4 s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, qh[n][b], zero, 0, 0, 0);
                        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, ql[n][b], s, 0, 0, 0);
#pragma unroll
                        for (int v = 0; v < 4; ++v) x[n][4 * u + v] = fmaf(d[v], s[v], x[n][4 * u + v]);
                    }
                }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    f32x4 sh = zero, sl = zero;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        sh = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[u * NB + b], qh[n][b], sh, 0, 0, 0);
                        sl = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[u * NB + b], ql[n][b], sl, 0, 0, 0);
                    }
#pragma unroll
                    for (int v = 0; v < 4; ++v) x[n][4 * u + v] = sh[v] + sl[v];
                }
        }
        const bool full = !meta && !(SHAPED && a.mask) && t * TK + TK - 1 <= wmin && t * TK + TK - 1 < a.T;
        h8 ph[NR][TT], pl[NR][TT];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            if constexpr (SHAPED) {
#pragma unroll
                for (int v = 0; v < U * 4; ++v) x[n][v] *= c[n];
                if (shape.cap > 0.0f) {
#pragma unroll
                    for (int v = 0; v < U * 4; ++v) x[n][v] = shape.cap * tanhFit(x[n][v] * shape.inv_cap);
                }
#pragma unroll
                for (int v = 0; v < U * 4; ++v) {
                    const int key = t * TK + 16 * (v >> 2) + 4 * kg + (v & 3);
                    const bool in = key < a.T;
                    int p = in ? key : kNoKey, dd = 0;
                    if (in && kpos) {
                        p = kpos[key];
                        if (p < 0) p = kNoKey;
                    }
                    if (in && kdoc) dd = kdoc[key];
                    if (shape.bias) x[n][v] = fmaf(-row[n].slope, fabsf((float)(row[n].pos - p)), x[n][v]);
                    if (a.mask && in) x[n][v] = addMask(x[n][v], a.mask[(size_t)row[n].token * a.m_row2 + key]);
                    x[n][v] = p <= row[n].limit && dd == row[n].doc ? x[n][v] * kLog2e : -INFINITY;
                }
            } else {
                const float c2 = c[n] * kLog2e;
#pragma unroll
                for (int v = 0; v < U * 4; ++v) x[n][v] *= c2;
                if (!full) {
                    const int last = min(row[n].limit, a.T - 1) - t * TK - 4 * kg;
#pragma unroll
                    for (int v = 0; v < U * 4; ++v) x[n][v] = 16 * (v >> 2) + (v & 3) <= last ? x[n][v] : -INFINITY;
                }
            }
            float bm = x[n][0];
#pragma unroll
            for (int v = 1; v < U * 4; ++v) bm = fmaxf(bm, x[n][v]);
            bm = fmaxf(bm, __shfl_xor(bm, 16));
            bm = fmaxf(bm, __shfl_xor(bm, 32));
            const float mn = fmaxf(m[n], bm), ms = mn == -INFINITY ? 0.0f : mn;
            if (__any(mn > m[n])) {
                const float alpha = ex2(m[n] - ms);
                l[n] *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[n][d] *= alpha;
                m[n] = mn;
            }
#pragma unroll
            for (int v = 0; v < U * 4; ++v) {
                x[n][v] = ex2(x[n][v] - ms);
                l[n] += x[n][v];
                const float ps = x[n][v] * kP;
                const _Float16 hi = (_Float16)ps;
                ph[n][v >> 3][v & 7] = hi;
                pl[n][v >> 3][v & 7] = (_Float16)(ps - (float)hi);
            }
        }
        if (__builtin_expect(__any(wild), 0)) {  // values that are no matrix operands, for the rows that see them
#pragma unroll 1
            for (int key = 0; key < TK; ++key) {
                const char* vrow = vb + (size_t)min(t * TK + key, a.T - 1) * a.v_row;
                const int xi = 4 * (key >> 4) + (key & 3), from = i + 16 * ((key >> 2) & 3);
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    const float p = __shfl(pick<U * 4>(x[n], xi), from) * kP;
                    if (!__any(p != 0.0f)) continue;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            const int rr = 4 * kg + v;
                            const float z = wildValue<Q4>(vrow, Q4 ? 32 * (d >> 1) + 8 * (d & 1) + (rr >> 1) + 16 * (rr & 1) : 16 * d + rr);
                            if (p != 0.0f && z != 0.0f) o[n][d][v] = fmaf(p, z, o[n][d][v]);
                        }
                }
            }
        }
        if constexpr (Q4) {
            const unsigned short* vd = reinterpret_cast<const unsigned short*>(mine + G::oD);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                h8 dh[2], dl[2];
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    dh[w] = *reinterpret_cast<const h8*>(vd + ((b * 2 + w) * 4 + kg) * 8);
                    dl[w] = *reinterpret_cast<const h8*>(vd + 64 * NB + ((b * 2 + w) * 4 + kg) * 8);
                }
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int d = 2 * b + s;
                    const i2 w2 = __builtin_amdgcn_ds_read_tr4_b64_v2i32((LdsI2)(mine + G::oV + trow * G::Row + 8 * d));
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const h8 code = nibbles((uint32_t)w2[w]);
                        const h8 vh = code * dh[w], vl = code * dl[w];
#pragma unroll
                        for (int n = 0; n < NR; ++n) {
                            o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, ph[n][w], o[n][d], 0, 0, 0);
                            o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, pl[n][w], o[n][d], 0, 0, 0);
                            o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph[n][w], o[n][d], 0, 0, 0);
                        }
                    }
                }
            }
        } else {
            const _Float16* vcol = reinterpret_cast<const _Float16*>(mine) + (4 * kg + (i >> 2)) * (G::VRow / 2) + 4 * (i & 3);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const s4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(vcol + 16 * d));
                const s4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(vcol + 16 * d + 16 * (G::VRow / 2)));
                const h8 va = __builtin_bit_cast(h8, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[n][0], o[n][d], 0, 0, 0);
                    o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[n][0], o[n][d], 0, 0, 0);
                }
            }
        }
        waveLds();
    }

    // ---- the four wavefronts' results joined, in their order
    __syncthreads();
    float* jo = reinterpret_cast<float*>(lds);
    float* jm = jo + 4 * NR * 16 * G::ORow;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
        const int at = (wave * NR + n) * 16 + i;
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(jo + at * G::ORow + 16 * d + 4 * kg) = o[n][d];
        if (kg == 0) {
            jm[2 * at] = m[n];
            jm[2 * at + 1] = l[n];
        }
    }
    __syncthreads();
    const int total = a.rows * D;
    for (int x = tid; x < total; x += 256) {
        const int r = x / D, at = x % D;
        float M = -INFINITY, f[4], L = 0.0f, y = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, jm[2 * (w * NR * 16 + r)]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float mw = jm[2 * (w * NR * 16 + r)];
            f[w] = mw == -INFINITY ? 0.0f : ex2(mw - M);
            L = fmaf(f[w], jm[2 * (w * NR * 16 + r) + 1], L);
            if (f[w] != 0.0f) y = fmaf(f[w], jo[(w * NR * 16 + r) * G::ORow + at], y);
        }
        const int b = at >> 5, rr = at & 15, dd = Q4 ? 32 * b + 8 * ((at >> 4) & 1) + (rr >> 1) + 16 * (rr & 1) : at;
        if (a.splits == 1) {
            const int token = r / a.G, head = kvh * a.G + (r - token * a.G);
            a.out[((size_t)token * a.H + head) * D + dd] = L == 0.0f ? 0.0f : y * (1.0f / (L * kP));
            if (a.lse && at == 0) a.lse[(size_t)token * a.H + head] = L == 0.0f ? -INFINITY : fmaf(M, kLn2, logf(L));
        } else {
            float* dst = a.part + (((size_t)sp * a.H_kv + kvh) * a.rows + r) * (D + 2);
            dst[dd] = y * (1.0f / kP);
            if (at == 0) {
                dst[D] = M;
                dst[D + 1] = L;
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------- joining key ranges
// One workgroup per row: o = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), the ranges dealt to four wavefronts whose sums are
// added in order. What counts is the latency of two dependent loads.
template <int D>
__global__ __launch_bounds__(256) void flash_ext_join_kernel(FxParams a) {
    constexpr int V = D / 64;
    __shared__ float sum[4][D];
    const int r = blockIdx.x, kvh = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t step = (size_t)a.H_kv * a.rows * (D + 2);
    const float* base = a.part + ((size_t)kvh * a.rows + r) * (D + 2);
    float M = -INFINITY;
    for (int s = lane; s < a.splits; s += 64) M = fmaxf(M, base[s * step + D]);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) M = fmaxf(M, __shfl_xor(M, x));
    float L = 0.0f;
    for (int s = lane; s < a.splits; s += 64) {
        const float ms = base[s * step + D];
        L += ms == -INFINITY ? 0.0f : ex2(ms - M) * base[s * step + D + 1];
    }
#pragma unroll
    for (int x = 1; x < 64; x *= 2) L += __shfl_xor(L, x);
    float y[V] = {};
#pragma unroll 4
    for (int s = wave; s < a.splits; s += 4) {
        const float ms = base[s * step + D], f = ms == -INFINITY ? 0.0f : ex2(ms - M);
#pragma unroll
        for (int x = 0; x < V; ++x) {
            const float z = base[s * step + lane + 64 * x];
            y[x] = f != 0.0f ? fmaf(f, z, y[x]) : y[x];
        }
    }
#pragma unroll
    for (int x = 0; x < V; ++x) sum[wave][lane + 64 * x] = y[x];
    __syncthreads();
    const int token = r / a.G, head = kvh * a.G + (r - token * a.G);
    for (int x = threadIdx.x; x < D; x += 256) {
        const float z = sum[0][x] + sum[1][x] + sum[2][x] + sum[3][x];
        a.out[((size_t)token * a.H + head) * D + x] = L == 0.0f ? 0.0f : z * (1.0f / L);
    }
    if (a.lse && threadIdx.x == 0) a.lse[(size_t)token * a.H + head] = L == 0.0f ? -INFINITY : fmaf(M, kLn2, logf(L));
}

template <class F>
int allow(F* kernel, int lds) {
    return fromHip(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds),
                   "flash_ext: LDS size");
}

template <int D, bool Q4, bool SHAPED>
int run(const FxParams& p, const FxPlan& plan, hipStream_t s) {
    if (plan.few) {
        const dim3 grid(p.splits, p.H_kv);
        constexpr int NR2 = D == 256 ? 1 : 2;  // (fxPlan: no more than 16 rows of 256)
        if (p.rows <= 16) {
            constexpr int lds = FewGeo<D, Q4, 1>::Lds;
            static const int ok = allow(flash_ext_few_kernel<D, Q4, SHAPED, 1>, lds);
            if (ok) return ok;
            hipLaunchKernelGGL((flash_ext_few_kernel<D, Q4, SHAPED, 1>), grid, dim3(256), lds, s, p);
        } else {
            constexpr int lds = FewGeo<D, Q4, NR2>::Lds;
            static const int ok = allow(flash_ext_few_kernel<D, Q4, SHAPED, NR2>, lds);
            if (ok) return ok;
            hipLaunchKernelGGL((flash_ext_few_kernel<D, Q4, SHAPED, NR2>), grid, dim3(256), lds, s, p);
        }
    } else {
        constexpr int lds = Geo<D, Q4>::Lds;
        static const int ok = allow(flash_ext_kernel<D, Q4, SHAPED>, lds);
        if (ok) return ok;
        hipLaunchKernelGGL((flash_ext_kernel<D, Q4, SHAPED>), dim3(p.H_kv, (p.rows + 127) / 128, p.splits), dim3(256), lds, s, p);
    }
    if (int e = fromHip(hipGetLastError(), "flash_ext")) return e;
    if (p.splits > 1) {
        hipLaunchKernelGGL(flash_ext_join_kernel<D>, dim3(p.rows, p.H_kv), dim3(256), 0, s, p);
        return fromHip(hipGetLastError(), "flash_ext (join)");
    }
    return 0;
}

template <int D>
int runD(bool q4, bool shaped, const FxParams& p, const FxPlan& plan, hipStream_t s) {
    if (q4) return shaped ? run<D, true, true>(p, plan, s) : run<D, true, false>(p, plan, s);
    return shaped ? run<D, false, true>(p, plan, s) : run<D, false, false>(p, plan, s);
}

}  // namespace

int launchFlashExt(bool q4, const kcFlashExtArgs& a, hipStream_t s) {
    if (a.d.N == 0) return 0;
    FxParams p = fxParams(a.d, a.q, a.k, a.mask, a.qpos, a.kpos, a.qdoc, a.kdoc, a.slopes, a.scale, a.softcap);
    const FxPlan plan = fxPlan(a.d);
    p.v = static_cast<const char*>(a.v);
    p.out = a.out;
    p.lse = a.lse;
    p.part = a.part;
    p.splits = plan.splits;
    p.per = plan.per;
    const bool shaped = a.mask || a.kpos || a.kdoc || a.slopes || a.softcap > 0.0f;
    switch (a.d.D) {
        case 64: return runD<64>(q4, shaped, p, plan, s);
        case 128: return runD<128>(q4, shaped, p, plan, s);
        case 256: return runD<256>(q4, shaped, p, plan, s);
        default: return fromHip(hipErrorInvalidValue, "flash_ext: D");
    }
}

}  // namespace kcamd
