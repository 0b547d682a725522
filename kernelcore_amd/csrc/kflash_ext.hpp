// kflash_ext.hpp -- parameters and launchers of the attention kernels over a key/value cache (kflash_ext.hip: flash_ext_f16 /
// flash_ext_q4_0; kattn_weights.hip: attn_weights_f16 / attn_weights_q4_0).
#pragma once

#include <hip/hip_runtime.h>
#include <kernelcore/llm_kernels.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace kcamd {

struct FxParams {
    const float* q;
    const char* k;
    const char* v;
    const unsigned short* mask;
    const int *qpos, *kpos, *qdoc, *kdoc;
    const float* slopes;
    float* out;
    float* lse;
    float* part;
    const float* w_in;  // attn_weights
    float* w;
    long long k_row, k_head, v_row, v_head, m_row2;  // (m_row2: fp16 values between mask rows, past 32 bits for rows 4 GiB apart)
    int H, H_kv, G, N, T, q_tok, q_head, key_row, pos0, causal, prefix, rows;
    int splits;  // key ranges
    int w_row;
    float scale, softcap, decay;
};

// How flash_ext splits a call. The few-rows kernel takes groups of 32 rows (16 of 256 values, beyond which it runs out of
// registers), the many-rows kernel blocks of 128; the keys go to `splits` ranges in turn. One group always runs on the
// few-rows kernel, several while they leave a compute unit no more than four units of keys (128 values; eight otherwise): 64 tokens over 500
// positions, 32 heads of 128 on 8, fp16: 14.3 us, on the many-rows kernel 18.0; over 8191: 9 tokens 26.4 and 20.3; 9 tokens over
// 2048, heads of 256: 20.6 and 35.9.
struct FxPlan {
    bool few;
    int splits;
    int64_t partFloats;
};
// Key ranges of the many-rows kernel, of four units at least: the least estimate, in steps (64 keys in 2 us, of 256 values 32 in 3.5).
// A compute unit holds one workgroup, which takes four steps to set up and write; ranges are written and read again by the join.
// Causal rows' workgroups, the longest first, fill the GPU evenly as they are, and are divided only where they do not fill it; equal
// ones run in whole rounds. 300 tokens over 3577: three ranges 55 us, six 73, two 67; 500 tokens over themselves: one 22.6, two
// 28.1; 82 over 3169: ten 30.1, thirteen 40.2; 1500 over 3000: one 88, two 98.
inline int64_t fxRanges(const kcFlashExtDims& d, int64_t base, int64_t units) {
    const double steps = d.D == 256 ? 2.0 * units : 1.0 * units;
    const double join = double(d.N) * d.H * d.D * 8 / 4.75e12 / (d.D == 256 ? 3.5e-6 : 2e-6);
    const int64_t most = std::min<int64_t>((units + 3) / 4, std::max<int64_t>(1, (d.causal ? 256 : 1024) / std::max<int64_t>(1, base)));
    int64_t best = 1;
    double least = 0.0;
    for (int64_t s = 1; s <= std::min<int64_t>(most, 256); ++s) {
        const double rounds = std::ceil(double(base) * s / 256.0);
        const double cost = rounds * (std::ceil(steps / s) + 4.0) + (s > 1 ? 2.0 + s * join : 0.0);
        if (s == 1 || cost < least) {
            best = s;
            least = cost;
        }
    }
    return best;
}
inline FxPlan fxPlan(const kcFlashExtDims& d) {
    const int64_t rows = int64_t(d.N) * (d.H / d.H_kv), units = (int64_t(d.T) + 63) / 64;
    const int64_t group = d.D == 256 ? 16 : 32, groups = (rows + group - 1) / group;
    FxPlan p{groups <= 1 || d.H_kv * groups * std::max<int64_t>(1, units) <= (d.D == 128 ? 1024 : 2048), 1, 0};
    const int64_t base = int64_t(d.H_kv) * (p.few ? groups : (rows + 127) / 128);
    // few rows: ranges of two units while that is no more than a workgroup for each of the 256 compute units (a wavefront then
    // has one tile of an fp16 cache), of four beyond, up to two workgroups each; T 2049, 5 tokens: 17 ranges 13.3 us, 9 14.6;
    // T 8191, 1 token: 64 ranges 14.2 us, 32 12.1
    const int64_t one = std::max<int64_t>(1, 256 / std::max<int64_t>(1, base)), two = std::max<int64_t>(1, 512 / std::max<int64_t>(1, base));
    int64_t splits = p.few ? std::max(std::min(two, (units + 3) / 4), std::min(one, (units + 1) / 2)) : fxRanges(d, base, units);
    p.splits = int(std::max<int64_t>(1, splits));
    p.partFloats = p.splits > 1 ? int64_t(p.splits) * d.H_kv * rows * (d.D + 2) : 0;
    return p;
}

int launchFlashExt(bool q4, const kcFlashExtArgs& a, hipStream_t s);
int launchAttnWeights(bool q4, const kcAttnWeightsArgs& a, hipStream_t s);

// The kernels' parameters of checked arguments.
inline FxParams fxParams(const kcFlashExtDims& d, const float* q, const void* k, const int* mask, const int* qpos,
                         const int* kpos, const int* qdoc, const int* kdoc, const float* slopes, float scale,
                         float softcap) {
    FxParams p{};
    p.q = q;
    p.k = static_cast<const char*>(k);
    p.mask = reinterpret_cast<const unsigned short*>(mask);
    p.qpos = qpos;
    p.kpos = kpos;
    p.qdoc = qdoc;
    p.kdoc = kdoc;
    p.slopes = slopes;
    p.k_row = d.k_row;
    p.k_head = d.k_head;
    p.v_row = d.v_row;
    p.v_head = d.v_head;
    p.H = d.H;
    p.H_kv = d.H_kv;
    p.G = d.H / d.H_kv;
    p.N = d.N;
    p.T = d.T;
    p.q_tok = d.q_tok;
    p.q_head = d.q_head;
    p.m_row2 = 2ll * d.m_row;
    p.key_row = d.key_row;
    p.pos0 = d.pos0;
    p.causal = d.causal;
    p.prefix = d.prefix;
    p.rows = d.N * p.G;
    p.scale = scale;
    p.softcap = softcap;
    return p;
}

}  // namespace kcamd
