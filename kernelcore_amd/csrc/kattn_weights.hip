// kattn_weights.hip -- attn_weights_f16 / attn_weights_q4_0 (gfx950): what the query rows gave each cached position,
//   w_gj = decay w_in_gj + sum over rows r of KV head g of exp(x_rj - lse_r)
// with x as flash_ext computes it (kflash_ext.hpp). Tiles of 32 keys x 32 rows on the matrix cores, S^T = K Q^T; a wavefront
// keeps its key tile and walks over the rows, each lane adding up its own row's weights for its 16 keys, so that the sum over
// the lanes is taken once, at the end, in one order. Four wavefronts share a tile's rows, or take tiles of their own where
// there are few rows: a single token's call reads K once and is bound by that.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "internal.hpp"
#include "kflash_ext_device.hpp"

namespace kcamd {
namespace {

using namespace fx;

template <int D, bool Q4>
struct WGeo {
    static constexpr int NB = D / 32;
    static constexpr int oS = 32 * kKeyRow<D>, oMeta = oS + (Q4 ? NB * 128 : 0), Tile = oMeta + 256;
};

// RW wavefronts per key tile (1, 2 or 4), 4 / RW tiles per workgroup.
template <int D, bool Q4, int RW>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attn_weights_kernel(FxParams a) {
    using G = WGeo<D, Q4>;
    constexpr int NB = G::NB, KT = 4 / RW, GT = 64 * RW;
    extern __shared__ int4 lds4[];
    __shared__ float part[4][32];
    const int kvh = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31, h = lane >> 5;
    const int kt = wave / RW, rw = wave % RW, gt = tid % GT;
    const int t = blockIdx.x * KT + kt;
    char* tile = reinterpret_cast<char*>(lds4) + kt * G::Tile;
    const char* kb = a.k + (size_t)kvh * a.k_head;
    const int* kpos = a.kpos ? a.kpos + (size_t)kvh * a.key_row : nullptr;
    const int* kdoc = a.kdoc ? a.kdoc + (size_t)kvh * a.key_row : nullptr;
    const bool meta = kpos || kdoc;
    const bool have = (long long)t * 32 < a.T;
    if (have) {
        if constexpr (Q4) {
            for (int i = gt; i < 32 * NB; i += GT) {
                const int key = i / NB, b = i % NB;
                const char* p = kb + (size_t)min(t * 32 + key, a.T - 1) * a.k_row + 18 * b;
                const u4 raw = *reinterpret_cast<const u4a2*>(p + 2);
                h8 code[4];
                blockCodes(raw, code);
                h8* dst = reinterpret_cast<h8*>(tile + key * kKeyRow<D> + 64 * b);
#pragma unroll
                for (int e = 0; e < 4; ++e) dst[e] = code[e];
                reinterpret_cast<float*>(tile + G::oS)[b * 32 + key] = halfBits(loadHalf(p));
            }
        } else {
            for (int i = gt; i < 32 * (D / 8); i += GT) {
                const int key = i / (D / 8), ch = i % (D / 8);
                *reinterpret_cast<u4*>(tile + key * kKeyRow<D> + 16 * ch) =
                    *reinterpret_cast<const u4a4*>(kb + (size_t)min(t * 32 + key, a.T - 1) * a.k_row + 16 * ch);
            }
        }
        if (meta && gt < 64) {
            const int key = t * 32 + (gt & 31);
            int x;
            if (gt < 32) {
                x = key < a.T ? (kpos ? kpos[key] : key) : kNoKey;
                if (x < 0) x = kNoKey;
            } else {
                x = kdoc && key < a.T ? kdoc[key] : 0;
            }
            reinterpret_cast<int*>(tile + G::oMeta)[gt] = x;
        }
    }
    __syncthreads();
    float acc[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0.0f;
    const Shape shape = shapeOf(a);
    for (int r0 = 32 * rw; have && r0 < a.rows; r0 += 32 * RW) {
        const Row row = rowOf(a, kvh, r0 + j);
        const int wmax = waveMax(row.live ? row.limit : -1);
        if (!kpos && t * 32 > wmax) continue;
        h8 qh[D / 16], ql[D / 16];
        const float c = loadRow32<D>(a, row, h, qh, ql);
        const float lse = row.live ? a.lse[(size_t)row.token * a.H + row.head] : -INFINITY;
        const unsigned short* mrow = a.mask ? a.mask + (size_t)row.token * a.m_row2 : nullptr;
        MaskWords mk;
        if (mrow) mk.load(mrow, t, h, a.T);
        float x[16];
        keyScores<D, Q4>(tile, tile + G::oS, j, h, qh, ql, x);
        shapeScores(x, c, shape, row, meta ? reinterpret_cast<const int*>(tile + G::oMeta) : nullptr, mrow ? &mk : nullptr, t, h);
        const int last = meta ? INT_MAX : min(row.limit, a.T - 1) - t * 32 - 4 * h;
        const float l2 = lse * kLog2e;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const float p = 8 * (v >> 2) + (v & 3) <= last && x[v] != -INFINITY ? ex2(x[v] - l2) : 0.0f;
            acc[v] += lse == -INFINITY ? 0.0f : p;
        }
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) {
#pragma unroll
        for (int o = 1; o < 32; o *= 2) acc[v] += __shfl_xor(acc[v], o);
        if (j == 0) part[wave][8 * (v >> 2) + 4 * h + (v & 3)] = acc[v];
    }
    __syncthreads();
    if (tid < 32 * KT) {
        const int g = tid >> 5, key = (blockIdx.x * KT + g) * 32 + (tid & 31);
        if (key < a.T) {
            float s = part[g * RW][tid & 31];
#pragma unroll
            for (int x = 1; x < RW; ++x) s += part[g * RW + x][tid & 31];
            const size_t at = (size_t)kvh * a.w_row + key;
            a.w[at] = a.w_in ? fmaf(a.decay, a.w_in[at], s) : s;
        }
    }
}

template <int D, bool Q4, int RW>
int run(const FxParams& p, hipStream_t s) {
    constexpr int lds = WGeo<D, Q4>::Tile * (4 / RW);
    static const int ok = fromHip(hipFuncSetAttribute(reinterpret_cast<const void*>(attn_weights_kernel<D, Q4, RW>),
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, lds), "attn_weights: LDS size");
    if (ok) return ok;
    const int tiles = p.T / 32 + (p.T % 32 != 0), kt = 4 / RW;
    hipLaunchKernelGGL((attn_weights_kernel<D, Q4, RW>), dim3((tiles + kt - 1) / kt, p.H_kv), dim3(256), lds, s, p);
    return fromHip(hipGetLastError(), "attn_weights");
}

template <int D, bool Q4>
int runRows(const FxParams& p, hipStream_t s) {
    if (p.rows <= 32) return run<D, Q4, 1>(p, s);
    if (p.rows <= 64) return run<D, Q4, 2>(p, s);
    return run<D, Q4, 4>(p, s);
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
