// krope_ext.hip -- rope_ext: rotary positions of q and k with the fp16 store of k and v into cache rows; kcRopeFreqs on the host.
//
// y0 = x0 cos - x1 sin, y1 = x0 sin + x1 cos for the pairs of a head's rotated part, angle 2 pi frac(pos f) with f in revolutions per
// position: the product and its fraction are taken in 64 bits (at position 2^20 a 32-bit angle is off by 2^-5), cosine and sine in 32.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "internal.hpp"
#include "kserve.hpp"

namespace kcamd {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f4a4 __attribute__((aligned(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef h4 h4a2 __attribute__((aligned(2)));

constexpr int kThreads = 256, kAhead = 2, kPairs = 1024;  // pairs of a workgroup's tokens
// Tokens of a launch that stores k and v, about: the search for repeated slots grows with their square. What a launch stores lies over what the
// one before it did, so that no launch looks for later ones' slots. (24 + 2 x 8 heads of 128: 16384 tokens 119 us, in one launch 140; 65536
// 500, in launches of 16384 570, in one 770; 262144 2.0 ms and 7.9. 8200 in two 51, in one 48; about 10000 alike.) Of q alone: what a launch's
// threads allow.
constexpr int kLaunch = 8192, kRest = 2048, kLaunchQ = 1 << 20;

struct RopeArgs {
    const float *q, *k, *v;
    const int* pos;
    const double* freqs;
    const long long* slots;
    float* q_out;
    char *k_cache, *v_cache;
    int n, H, H_kv, D, n_rot;
    int q_tok, q_head, k_tok, k_head, v_tok, v_head, out_tok, out_head, cache_rows;
    long long kc_row, kc_head, vc_row, vc_head;
    float scale;
    int q_tokens, kv_tokens, kv_blocks;  // tokens of a workgroup, workgroups for k and v (the first ones, which take longest)
};

// Eight values of a row: two groups of four that hold four pairs, or of its unturned part; na and nb of them are there. Neighbouring
// threads' groups lie side by side.
struct Unit {
    int a, b, na, nb, pa, pb;  // pa, pb: the groups' first pairs, -1 for unturned values
};
template <bool INTER>
__device__ __forceinline__ Unit unitOf(int u, int n_rot, int D) {
    const int half = n_rot / 2, turned = (half + 3) / 4;
    Unit x;
    if (u < turned && !INTER) {
        x.pa = x.pb = 4 * u;
        x.a = 4 * u;
        x.b = x.a + half;
        x.na = x.nb = min(4, half - 4 * u);
    } else {
        const int from = u < turned ? 0 : n_rot, to = u < turned ? n_rot : D, y = u < turned ? u : u - turned;
        x.a = from + 4 * y;
        x.b = x.a + 4 * ((to - from + 7) / 8);
        x.na = min(4, to - x.a);
        x.nb = max(0, min(4, to - x.b));
        x.pa = u < turned ? x.a / 2 : -1;
        x.pb = x.b / 2;
    }
    return x;
}

template <bool FULL>
__device__ __forceinline__ f32x4 loadPart(const float* p, int n) {
    if (FULL || n == 4) return *reinterpret_cast<const f4a4*>(p);
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) x[e] = p[e];
    return x;
}
template <bool FULL>
__device__ __forceinline__ void storePart(float* p, f32x4 x, int n) {
    if (FULL || n == 4) {
        *reinterpret_cast<f4a4*>(p) = x;
        return;
    }
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) p[e] = x[e];
}
template <bool FULL>
__device__ __forceinline__ void storePart(_Float16* p, f32x4 x, int n) {
    if (FULL || n == 4) {
        *reinterpret_cast<h4a2*>(p) = h4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
        return;
    }
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < n) p[e] = (_Float16)x[e];
}

// (cs: the token's cosines and sines)
template <bool INTER>
__device__ __forceinline__ void turn(f32x4& a, f32x4& b, const Unit& u, const float2* cs, int pairs) {
    float2 z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = cs[min(INTER && e >= 2 ? u.pb + e - 2 : u.pa + e, pairs - 1)];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f32x4& lo = INTER ? (e < 2 ? a : b) : a;
        f32x4& hi = INTER ? (e < 2 ? a : b) : b;
        const int i = INTER ? 2 * (e & 1) : e, j = INTER ? i + 1 : e;
        const float x0 = lo[i], x1 = hi[j];
        lo[i] = fmaf(x0, z[e].x, -(x1 * z[e].y));
        hi[j] = fmaf(x0, z[e].y, x1 * z[e].x);
    }
}

// A workgroup takes all heads of q, or all of k and v, of q_tokens or kv_tokens tokens, eight values a thread at a time. The first kAhead
// of a thread's are loaded before the angles are computed (once, into LDS) and repeated slots looked for: what bounds it is the
// bytes, and for few tokens the latency of one load and the angles. 3333 tokens of 24 + 2 x 8 heads of 128, from memory: 27 us, 4.5 TB/s
// where a copy of as many bytes reaches 5.0 (35 us with loads after the angles and k and v last); one token 4 us.
// FULL: every group has its four values (heads and rotated parts of whole eights), so that a load is one and none waits for another (the prompt
// below 27 us, 28 without).
template <bool INTER, bool FULL>
__global__ __launch_bounds__(kThreads) void rope_ext_kernel(RopeArgs a) {
    __shared__ float2 cs[kPairs];
    __shared__ int later[16], rowOf[16];
    const int tid = threadIdx.x;
    const bool isQ = (int)blockIdx.x >= a.kv_blocks;
    const int per = isQ ? a.q_tokens : a.kv_tokens;
    const int t0 = (isQ ? blockIdx.x - a.kv_blocks : blockIdx.x) * per, n = min(per, a.n - t0);
    const int pairs = a.n_rot / 2;
    const int turned = (pairs + 3) / 4, units = turned + (a.D - a.n_rot + 7) / 8, vunits = (a.D + 7) / 8;
    const int heads = isQ ? a.H : a.H_kv, first = n * heads * units, all = first + (!isQ && a.v ? n * heads * vunits : 0);
    // where the x-th eight values are
    struct Place {
        const float* src;
        Unit u;
        int t, h;
        bool isV;
    };
    auto placeOf = [&](int x) {
        Place p;
        p.isV = x >= first;
        const int y = p.isV ? x - first : x, uu = p.isV ? vunits : units, row = y / uu;
        p.t = row / heads;
        p.h = row - p.t * heads;
        p.u = unitOf<INTER>(y - row * uu, p.isV ? 0 : a.n_rot, a.D);
        p.src = isQ ? a.q + (long long)(t0 + p.t) * a.q_tok + (long long)p.h * a.q_head
              : p.isV ? a.v + (long long)(t0 + p.t) * a.v_tok + (long long)p.h * a.v_head
                      : a.k + (long long)(t0 + p.t) * a.k_tok + (long long)p.h * a.k_head;
        return p;
    };
    Place at[kAhead];
    f32x4 lo[kAhead], hi[kAhead];
    auto load = [&](int x0) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int x = min(x0 + kThreads * k, all - 1);
            at[k] = placeOf(x);
            lo[k] = loadPart<FULL>(at[k].src + at[k].u.a, at[k].u.na);
            hi[k] = loadPart<FULL>(at[k].src + at[k].u.b, at[k].u.nb);
        }
    };
    load(tid);
    if (!isQ && tid < 16) {
        later[tid] = 0;
        const long long slot = tid < n ? a.slots[t0 + tid] : -1;
        rowOf[tid] = slot >= 0 && slot < a.cache_rows ? (int)slot : -1;
    }
    for (int x = tid; x < n * pairs; x += kThreads) {
        const int t = x / pairs, i = x - t * pairs;
        const double r = (double)a.pos[t0 + t] * a.freqs[i];
        const float f = 2.0f * (float)(r - rint(r));
        cs[x] = make_float2(cospif(f) * a.scale, sinpif(f) * a.scale);
    }
    __syncthreads();
    if (!isQ) {
        // tokens whose slot a later one repeats are left to that one
        for (int x = t0 + 1 + tid; x < a.n; x += kThreads) {
            const long long slot = a.slots[x];
            if (slot < 0 || slot >= a.cache_rows) continue;
            for (int t = 0; t < n; ++t)
                if (t0 + t < x && rowOf[t] == (int)slot) later[t] = 1;
        }
        __syncthreads();
    }
    for (int x0 = tid; x0 < all; x0 += kThreads * kAhead) {
        if (x0 != tid) load(x0);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (x0 + kThreads * k >= all) break;
            const Unit& u = at[k].u;
            const int t = at[k].t, h = at[k].h;
            if (u.pa >= 0) turn<INTER>(lo[k], hi[k], u, cs + t * pairs, pairs);
            if (isQ) {
                float* dst = a.q_out + (long long)(t0 + t) * a.out_tok + (long long)h * a.out_head;
                storePart<FULL>(dst + u.a, lo[k], u.na);
                storePart<FULL>(dst + u.b, hi[k], u.nb);
            } else if (rowOf[t] >= 0 && !later[t]) {
                char* to = at[k].isV ? a.v_cache + rowOf[t] * a.vc_row + h * a.vc_head : a.k_cache + rowOf[t] * a.kc_row + h * a.kc_head;
                _Float16* dst = reinterpret_cast<_Float16*>(to);
                storePart<FULL>(dst + u.a, lo[k], u.na);
                storePart<FULL>(dst + u.b, hi[k], u.nb);
            }
        }
    }
}

}  // namespace

int launchRopeExt(const kcRopeExtArgs& a, hipStream_t s) {
    const int launches = a.k ? std::max(1, (a.n_tokens - kRest + kLaunch - 1) / kLaunch) : 1;
    const int each = std::min(kLaunchQ, (a.n_tokens + launches - 1) / launches);
    for (int at = 0; at < a.n_tokens; at += each) {
        const int n = std::min(each, a.n_tokens - at);
        RopeArgs p{a.q ? a.q + (long long)at * a.q_tok : nullptr, a.k ? a.k + (long long)at * a.k_tok : nullptr, a.v ? a.v + (long long)at * a.v_tok : nullptr,
                   a.pos + at, a.freqs, reinterpret_cast<const long long*>(a.slots) + (a.k ? at : 0), a.q ? a.q_out + (long long)at * a.out_tok : nullptr,
                   static_cast<char*>(a.k_cache), static_cast<char*>(a.v_cache), n, a.H, a.H_kv, a.D, a.n_rot, a.q_tok, a.q_head, a.k_tok, a.k_head,
                   a.v_tok, a.v_head, a.out_tok, a.out_head, a.cache_rows, a.kc_row, a.kc_head, a.vc_row, a.vc_head, a.scale, 1, 1, 0};
        // k and v: up to 16 tokens share the search for repeated slots, which reads all later tokens' slots, once there are four workgroups
        // for each CU (3333 tokens with three to a workgroup 28 us, with six 31, with one 33)
        const int most = std::max(1, std::min(16, kPairs / std::max(1, a.n_rot / 2)));
        p.kv_tokens = std::max(1, std::min(most, n / 1024));
        // q: what a workgroup loads ahead, likewise
        const int units = a.n_rot / 8 + (a.D - a.n_rot + 7) / 8;
        p.q_tokens = std::max(1, std::min({most, n / 512, kAhead * kThreads / std::max(1, a.H * units)}));
        const int qBlocks = a.q ? (n + p.q_tokens - 1) / p.q_tokens : 0;
        p.kv_blocks = a.k ? (n + p.kv_tokens - 1) / p.kv_tokens : 0;
        const dim3 grid(p.kv_blocks + qBlocks);
        if (grid.x == 0) return 0;
        const bool full = a.n_rot % 8 == 0 && a.D % 8 == 0;
        if (a.interleaved && full) hipLaunchKernelGGL((rope_ext_kernel<true, true>), grid, dim3(kThreads), 0, s, p);
        else if (a.interleaved) hipLaunchKernelGGL((rope_ext_kernel<true, false>), grid, dim3(kThreads), 0, s, p);
        else if (full) hipLaunchKernelGGL((rope_ext_kernel<false, true>), grid, dim3(kThreads), 0, s, p);
        else hipLaunchKernelGGL((rope_ext_kernel<false, false>), grid, dim3(kThreads), 0, s, p);
        if (int e = fromHip(hipGetLastError(), "rope_ext")) return e;
    }
    return 0;
}

}  // namespace kcamd

kcError_t kcRopeFreqs(const kcRopeScaling* r, const float* ff, double* freqs, float* scale) noexcept {
    if (!r || !freqs || !scale || r->n_rot <= 0 || r->n_rot % 2 || r->n_rot > 1024 || !(r->base > 1.0f) || !std::isfinite(r->base) ||
        !(r->factor > 0.0f) || !std::isfinite(r->factor) || r->yarn_ctx < 0 || !(r->beta_fast >= 0.0f) || !(r->beta_slow >= 0.0f) ||
        !std::isfinite(r->beta_fast) || !std::isfinite(r->beta_slow)) {
        kcamd::setDetail("rope: n_rot even, from 2 to 1024, base above 1, factor positive, yarn_ctx and betas not negative");
        return kc::Error::InvalidValue;
    }
    const int n = r->n_rot;
    for (int i = 0; ff && i < n / 2; ++i)
        if (!(ff[i] > 0.0f) || !std::isfinite(ff[i])) {
            kcamd::setDetail("rope: frequency factors are positive and finite");
            return kc::Error::InvalidValue;
        }
    constexpr double kTwoPi = 6.283185307179586;
    // the pair that turns beta times within the original context
    const auto pairOf = [&](double beta) { return n * std::log(r->yarn_ctx / (beta * kTwoPi)) / (2 * std::log((double)r->base)); };
    double low = 0, high = 0;
    if (r->yarn_ctx) {
        low = std::max(0.0, std::floor(pairOf(r->beta_fast > 0.0f ? r->beta_fast : 32.0)));
        high = std::min(n - 1.0, std::ceil(pairOf(r->beta_slow > 0.0f ? r->beta_slow : 1.0)));
    }
    for (int i = 0; i < n / 2; ++i) {
        const double theta = std::pow((double)r->base, -2.0 * i / n) / (ff ? (double)ff[i] : 1.0);
        const double slow = r->yarn_ctx ? std::min(1.0, std::max(0.0, (i - low) / std::max(0.001, high - low))) : 1.0;
        freqs[i] = (theta / r->factor * slow + theta * (1 - slow)) / kTwoPi;
    }
    *scale = r->yarn_ctx ? (float)(1 + 0.1 * std::log((double)r->factor)) : 1.0f;
    return kc::Error::Success;
}
