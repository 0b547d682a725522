// kv_cache.hip -- rows of a cache: set_rows_q4_0 / get_rows_q4_0 (4-bit blocks), kv_keep (which positions to keep by their
// accumulated weight) and kv_gather (the kept rows into other memory).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "internal.hpp"
#include "kv_cache.hpp"

namespace kcamd {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f4a4 __attribute__((aligned(4)));
typedef uint32_t u32a2 __attribute__((aligned(2)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ long long index64(const int* idx, long long i) {
    return (long long)(((unsigned long long)(unsigned)idx[2 * i + 1] << 32) | (unsigned)idx[2 * i]);
}

// ---------------------------------------------------------------------------------------------- 4-bit rows
// Eight lanes per block of 32 values, four values each; R rows per workgroup. Bound by the search for repeated indices, in which a workgroup
// reads those of all later rows, and by reading the f32 rows: 1777 rows of 1024 values 5.6 us, 1.3 TB/s; one row 1.7 us. The search
// grows with the square of the rows: 8192 rows 16 us, 32768 85 (1.6 TB/s), 131072 0.96 ms (0.6), 524280 14 ms.
// Code of x: floor(x / d + 8.5), d = xm / -8. With a = |d| and y = x sign(d) that is the largest c with (c - 8.5) a <= y:
// the product c' a of a half-integer and an f32 is rounded by the fma only after y is subtracted, so the sign of
// y - c' a is exact and settles a guess from the rounded quotient.
__device__ __forceinline__ int code4(float y, float a, float inv) {
    float c = fminf(fmaxf(floorf(y * inv + 8.5f), 0.0f), 15.0f);
    if (fmaf(8.5f - c, a, y) < 0.0f) c -= 1.0f;
    else if (fmaf(7.5f - c, a, y) >= 0.0f) c += 1.0f;
    return (int)fminf(fmaxf(c, 0.0f), 15.0f);
}

template <int R>
__global__ __launch_bounds__(256) void set_rows_q4_0_kernel(const float* __restrict__ src, const int* __restrict__ idx,
                                                            char* __restrict__ dst, int nb, int rows, int src_row,
                                                            int dst_rows, long long dst_row) {
    __shared__ unsigned later;
    const int r0 = blockIdx.y * R, tid = threadIdx.x;
    const int b = blockIdx.x * 32 + (tid >> 3), l = tid & 7;
    const bool live = b < nb;
    f32x4 x[R];
    long long at[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
        const int r = min(r0 + k, rows - 1);
        at[k] = index64(idx, r);
        x[k] = *reinterpret_cast<const f4a4*>(src + (size_t)r * src_row + 32 * min(b, nb - 1) + 4 * l);
    }
    // rows whose index a later row repeats are left to that row
    if (tid == 0) later = 0;
    __syncthreads();
    unsigned mine = 0;
    for (int i0 = r0 + 1 + tid; i0 < rows; i0 += 4 * 256) {  // four loads at a time (past the end the last row's again)
        long long other[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) other[n] = index64(idx, min(i0 + 256 * n, rows - 1));
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int k = 0; k < R; ++k)
                if (min(i0 + 256 * n, rows - 1) > r0 + k && other[n] == at[k]) mine |= 1u << k;
    }
    if (mine) atomicOr(&later, mine);
    __syncthreads();
    const unsigned skip = later;
#pragma unroll
    for (int k = 0; k < R; ++k) {
        if (r0 + k >= rows || (skip >> k & 1u) || at[k] < 0 || at[k] >= dst_rows) continue;  // (the same for the workgroup)
        // the value of largest magnitude, the first of several
        float m = 0.0f;
        int first = 32;
        bool wild = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float v = x[k][e];
            wild |= !(fabsf(v) < INFINITY);
            if (fabsf(v) > fabsf(m)) {
                m = v;
                first = 4 * l + e;
            }
        }
        auto with = [&](auto from) {
            const float m2 = __builtin_bit_cast(float, from(__builtin_bit_cast(int, m)));
            const int f2 = from(first);
            wild |= from((int)wild) != 0;
            if (fabsf(m2) > fabsf(m) || (fabsf(m2) == fabsf(m) && f2 < first)) {
                m = m2;
                first = f2;
            }
        };
        with([](int y) { return __builtin_amdgcn_update_dpp(y, y, 0xB1, 0xF, 0xF, false); });   // lane ^ 1
        with([](int y) { return __builtin_amdgcn_update_dpp(y, y, 0x4E, 0xF, 0xF, false); });   // ^ 2
        with([](int y) { return __builtin_amdgcn_update_dpp(y, y, 0x141, 0xF, 0xF, false); });  // the other four of eight
        const float d = m * -0.125f, up = fabsf(d) < 0x1p-100f ? 0x1p64f : 1.0f;  // (subnormal steps scaled: exact)
        const float a = fabsf(d) * up, inv = 1.0f / a;
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = wild || a == 0.0f ? 8 : code4((d < 0.0f ? -x[k][e] : x[k][e]) * up, a, inv);
            w |= (uint32_t)c << (8 * e);
        }
        w |= (uint32_t)__shfl_xor((int)w, 4) << 4;  // (lanes 0 .. 3: the codes of values 16 on in the high bits)
        if (live) {
            char* p = dst + (size_t)at[k] * dst_row + 18 * (size_t)b;
            if (l < 4) *reinterpret_cast<u32a2*>(p + 2 + 4 * l) = w;
            if (l == 4) *reinterpret_cast<unsigned short*>(p) = wild ? (unsigned short)0x7E00 : __builtin_bit_cast(unsigned short, (_Float16)d);
        }
    }
}

// Eight lanes per block, four values (16 bytes of y) each. 1777 rows of 1024 values 4.8 us, 1.7 TB/s of y, a row to a workgroup: an
// index, then its block, then the store; 32768 rows 25 us, 5.4 TB/s, by writing y.
__global__ __launch_bounds__(256) void get_rows_q4_0_kernel(const char* __restrict__ src, const int* __restrict__ idx,
                                                            float* __restrict__ y, int nb, int rows, int src_rows,
                                                            long long src_row) {
    const int b = blockIdx.x * 32 + (threadIdx.x >> 3), l = threadIdx.x & 7;
    if (b >= nb) return;
    for (int r = blockIdx.y; r < rows; r += gridDim.y) {
        const long long at = index64(idx, r);
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (at >= 0 && at < src_rows) {
            const char* p = src + (size_t)at * src_row + 18 * (size_t)b;
            const float d = (float)__builtin_bit_cast(_Float16, *reinterpret_cast<const unsigned short*>(p));
            const uint32_t w = *reinterpret_cast<const u32a2*>(p + 2 + 4 * (l & 3)) >> (l & 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = d * (float)((int)(w >> (8 * e) & 15u) - 8);
        }
        *reinterpret_cast<f4a4*>(y + (size_t)r * nb * 32 + 32 * b + 4 * l) = v;
    }
}

// ---------------------------------------------------------------------------------------------- positions to keep
// One workgroup per head. The weight of rank `want` among the free positions by a radix search from the top (digits of 11, 11
// and 10 bits over order-preserving codes), then the positions above it and the first of those equal to it, written
// in ascending order: each wavefront owns a contiguous piece of the row, so that ballots and one prefix over the
// wavefronts give every position its place. Up to R x 1024 positions are read once and held in registers through the five
// sweeps; longer rows (R = 0) are read by each sweep. A head has one compute unit, and the sweeps' instructions bound it: 16384
// positions 12.4 us (digits of 8 bits, a sweep more: 1.3 us more), 1500 positions 5.6 us, its barriers and the load. Over 32768
// the sweeps' loads count too, one at a time: 32768 positions 22 us, 65536 70, 131072 134.
constexpr int kKeepThreads = 1024, kKeepWaves = kKeepThreads / 64;

__device__ __forceinline__ uint32_t rankCode(float w) {  // ascending with w; -0 as 0; NaN first; never 0
    const uint32_t u = __builtin_bit_cast(uint32_t, w == 0.0f ? 0.0f : w);
    return w != w ? 1u : (u & 0x80000000u ? ~u : u | 0x80000000u);
}

// The sum over this lane and those below it, in registers: within rows of 16, then from row to row.
__device__ __forceinline__ unsigned scanUp(unsigned x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // from the lanes 1, 2, 4 and 8 below
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // lane 15 of a row to the odd row above it
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // lane 31 to the upper two
    return x;
}
// The sum of the counts of the wavefronts before `wave`.
__device__ __forceinline__ unsigned sumBelow(const u4* counts, int wave) {
    unsigned sum = 0;
#pragma unroll
    for (int x = 0; x < kKeepWaves; ++x) sum += x < wave ? counts[x / 4][x % 4] : 0u;
    return sum;
}

template <int R>
__global__ __launch_bounds__(kKeepThreads) void kv_keep_kernel(const float* __restrict__ w, int* __restrict__ keep, int T,
                                                               int w_row, int n_keep, int keep_row, int first, int recent) {
    __shared__ uint2 hist[2][kKeepThreads];  // of 2048 digits
    __shared__ unsigned found[2];
    __shared__ u4 waves[kKeepWaves / 4], above[kKeepWaves / 4], equal[kKeepWaves / 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float* wr = w + (size_t)blockIdx.x * w_row;
    int* out = keep + (size_t)blockIdx.x * keep_row;
    const int lo = first, hi = T - recent;      // the free positions
    unsigned want = n_keep - first - recent;    // how many of them stay
    const int piece = ((hi - lo + kKeepWaves - 1) / kKeepWaves + 63) / 64 * 64;
    const int p0 = (int)min((long long)hi, lo + (long long)wave * piece), p1 = min(hi, p0 + piece);
    const int n = (p1 - p0 + 63) / 64;          // (at most R where R > 0)
    uint32_t held[R > 0 ? R : 1];
    if constexpr (R > 0) {
        float x[R];
#pragma unroll
        for (int k = 0; k < R; ++k) x[k] = k < n ? wr[min(p0 + 64 * k + lane, p1 - 1)] : 0.0f;
#pragma unroll
        for (int k = 0; k < R; ++k) held[k] = p0 + 64 * k + lane < p1 ? rankCode(x[k]) : 0u;
    }
    // f(position, code) for this wavefront's positions, 64 at a time; code 0, less than any weight's, for the lanes past its piece
    auto sweep = [&](auto&& f) {
        if constexpr (R > 0) {
#pragma unroll
            for (int k = 0; k < R; ++k)
                if (k < n) f(p0 + 64 * k + lane, held[k]);
        } else {
            for (int k = 0; k < n; ++k) {
                const int i = p0 + 64 * k + lane;
                const uint32_t u = rankCode(wr[min(i, p1 - 1)]);
                f(i, i < p1 ? u : 0u);
            }
        }
    };
    for (int i = tid; i < first; i += kKeepThreads) out[i] = i;
    for (int i = tid; i < recent; i += kKeepThreads) out[n_keep - recent + i] = T - recent + i;
    if (want == 0) return;
    hist[0][tid] = make_uint2(0, 0);
    __syncthreads();

    uint32_t prefix = 0;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        constexpr int kShift[3] = {21, 10, 0};
        const int shift = kShift[pass], bits = pass < 2 ? 11 : 10;
        unsigned* digits = reinterpret_cast<unsigned*>(hist[pass & 1]);
        sweep([&](int, uint32_t u) {
            if (pass == 0 || u >> (shift + bits) == prefix) atomicAdd(digits + (u >> shift & ((1u << bits) - 1)), 1u);
        });
        if (pass < 2) hist[~pass & 1][tid] = make_uint2(0, 0);
        __syncthreads();
        // the digit at which the count from the top reaches `want`: two digits a thread
        const int d = kKeepThreads - 1 - tid;
        const uint2 c = hist[pass & 1][d];
        unsigned upto = c.x + c.y;
        upto = scanUp(upto);
        if (lane == 63) reinterpret_cast<unsigned*>(waves)[wave] = upto;
        __syncthreads();
        const unsigned before = upto - c.x - c.y + sumBelow(waves, wave);
        if (before < want && before + c.y >= want) {
            found[0] = 2 * d + 1;
            found[1] = want - before;
        } else if (before + c.y < want && before + c.y + c.x >= want) {
            found[0] = 2 * d;
            found[1] = want - before - c.y;
        }
        __syncthreads();
        prefix = prefix << bits | found[0];
        want = found[1];
    }
    // prefix: the code of the last weight that stays; want: how many equal to it stay
    int gt = 0, eq = 0;
    sweep([&](int, uint32_t u) {
        gt += (int)__popcll(__ballot(u > prefix));
        eq += (int)__popcll(__ballot(u == prefix));
    });
    if (lane == 0) {
        reinterpret_cast<unsigned*>(above)[wave] = gt;
        reinterpret_cast<unsigned*>(equal)[wave] = eq;
    }
    __syncthreads();
    int ties = (int)sumBelow(equal, wave), at = first + (int)sumBelow(above, wave) + min(ties, (int)want);  // of the pieces before this one
    const unsigned long long below = (1ull << lane) - 1;
    sweep([&](int i, uint32_t u) {
        const unsigned long long e = __ballot(u == prefix);
        const bool stays = u > prefix || (u == prefix && ties + (int)__popcll(e & below) < (int)want);
        const unsigned long long s = __ballot(stays);
        if (stays) out[at + (int)__popcll(s & below)] = i;
        at += (int)__popcll(s);
        ties += (int)__popcll(e);
    });
}

// ---------------------------------------------------------------------------------------------- kept rows
// One grid over planes, heads and rows. A row's units (the widest of 16, 8, 4 and 2 bytes that all addresses of a plane
// allow) lie on the next power of two of lanes, up to 256; each thread moves up to eight units whose loads are all in flight
// before the first store. Bound by memory: 4096 rows of 256 bytes of K and V and 8 heads 8.6 us, 3.9 TB/s read and written.
struct GatherPlane {
    const char* src;
    char* dst;
    long long src_row, src_head, dst_row, dst_head;
    int units, unit, lanes;  // units of a row, bytes of a unit, log2 of the lanes to a row
};
struct GatherArgs {
    GatherPlane p[4];
    const int* keep;
    int n_keep, keep_row, T;
};
constexpr int kGather = 8;

template <class U>
__device__ __forceinline__ void gatherRows(const GatherPlane& p, const int* keep, int n_keep, int T, int g) {
    const int per = 256 >> p.lanes, u0 = threadIdx.x & ((1 << p.lanes) - 1);  // rows of a pass, this thread's unit
    const long long r0 = (long long)blockIdx.x * per * kGather + (threadIdx.x >> p.lanes);
    if (r0 >= n_keep) return;
    const char* src = p.src + g * p.src_head;
    char* dst = p.dst + g * p.dst_head;
    int from[kGather];
#pragma unroll
    for (int k = 0; k < kGather; ++k) {
        from[k] = -1;
        if (r0 + per * k < n_keep) {
            const int s = keep[r0 + per * k];
            from[k] = s < T ? s : -1;
        }
    }
    for (int u = u0; u < p.units; u += 256) {  // (more than once only in rows of more than 256 units)
        U x[kGather];
#pragma unroll
        for (int k = 0; k < kGather; ++k)
            if (from[k] >= 0) x[k] = *reinterpret_cast<const U*>(src + (long long)from[k] * p.src_row + (long long)u * (int)sizeof(U));
#pragma unroll
        for (int k = 0; k < kGather; ++k)
            if (from[k] >= 0) *reinterpret_cast<U*>(dst + (r0 + per * k) * p.dst_row + (long long)u * (int)sizeof(U)) = x[k];
    }
}

__global__ __launch_bounds__(256) void kv_gather_kernel(GatherArgs a) {
    const GatherPlane& p = a.p[blockIdx.z];
    const int g = blockIdx.y;
    const int* keep = a.keep + (size_t)g * a.keep_row;
    if (p.unit == 16) gatherRows<u4>(p, keep, a.n_keep, a.T, g);
    else if (p.unit == 8) gatherRows<u2>(p, keep, a.n_keep, a.T, g);
    else if (p.unit == 4) gatherRows<uint32_t>(p, keep, a.n_keep, a.T, g);
    else gatherRows<unsigned short>(p, keep, a.n_keep, a.T, g);
}

}  // namespace

int launchSetRowsQ40(const kcSetRowsQ40Args& a, hipStream_t s) {
    if (a.rows == 0) return 0;
    const int nb = a.n / 32;
    char* dst = static_cast<char*>(a.dst);
    auto run = [&](auto kernel, int r) {
        hipLaunchKernelGGL(kernel, dim3((nb + 31) / 32, (a.rows + r - 1) / r), dim3(256), 0, s, a.src, a.idx, dst, nb, a.rows, a.src_row,
                           a.dst_rows, a.dst_row);
    };
    // rows of a workgroup share its search for repeated indices, which grows with the rows; few rows fill the GPU one each
    if (a.rows <= 2048) run(set_rows_q4_0_kernel<1>, 1);
    else if (a.rows <= 8192) run(set_rows_q4_0_kernel<2>, 2);
    else run(set_rows_q4_0_kernel<8>, 8);
    return fromHip(hipGetLastError(), "set_rows_q4_0");
}

int launchGetRowsQ40(const kcGetRowsQ40Args& a, hipStream_t s) {
    if (a.rows == 0) return 0;
    const int nb = a.n / 32;
    hipLaunchKernelGGL(get_rows_q4_0_kernel, dim3((nb + 31) / 32, std::min(a.rows, 4096)), dim3(256), 0, s,
                       static_cast<const char*>(a.src), a.idx, a.y, nb, a.rows, a.src_rows, a.src_row);
    return fromHip(hipGetLastError(), "get_rows_q4_0");
}

int launchKvKeep(const kcKvKeepArgs& a, hipStream_t s) {
    if (a.n_keep == 0) return 0;
    auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(a.heads), dim3(kKeepThreads), 0, s, a.w, a.keep, a.T, a.w_row, a.n_keep, a.keep_row, a.first,
                           a.recent);
    };
    // (a wavefront's piece is a sixteenth of the free positions, rounded up to 64: R 64 at most)
    if (a.T <= 5 * kKeepThreads - 1024) run(kv_keep_kernel<5>);
    else if (a.T <= 17 * kKeepThreads - 1024) run(kv_keep_kernel<17>);
    else if (a.T <= 33 * kKeepThreads - 1024) run(kv_keep_kernel<33>);
    else run(kv_keep_kernel<0>);
    return fromHip(hipGetLastError(), "kv_keep");
}

int launchKvGather(const kcKvGatherArgs& a, hipStream_t s) {
    if (a.n_keep == 0) return 0;
    GatherArgs g{};
    long long blocks = 1;
    for (int i = 0; i < a.n_planes; ++i) {
        const kcKvPlane& p = a.planes[i];
        const auto all = reinterpret_cast<uintptr_t>(p.src) | reinterpret_cast<uintptr_t>(p.dst) | uintptr_t(p.src_row) |
                         uintptr_t(p.src_head) | uintptr_t(p.dst_row) | uintptr_t(p.dst_head) | uintptr_t(p.bytes);
        const int unit = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2, units = p.bytes / unit;
        int lanes = 0;
        while (lanes < 8 && (1 << lanes) < units) ++lanes;
        g.p[i] = GatherPlane{static_cast<const char*>(p.src), static_cast<char*>(p.dst), p.src_row, p.src_head, p.dst_row,
                             p.dst_head, units, unit, lanes};
        const int rows = (256 >> lanes) * kGather;
        blocks = std::max(blocks, ((long long)a.n_keep + rows - 1) / rows);
    }
    g.keep = a.keep;
    g.n_keep = a.n_keep;
    g.keep_row = a.keep_row;
    g.T = a.T;
    hipLaunchKernelGGL(kv_gather_kernel, dim3((unsigned)blocks, a.heads, a.n_planes), dim3(256), 0, s, g);
    return fromHip(hipGetLastError(), "kv_gather");
}

}  // namespace kcamd
