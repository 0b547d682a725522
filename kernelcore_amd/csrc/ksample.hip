// ksample.hip -- sample_rows: temperature, top-k, top-p, min-p and the draw from given random numbers, without a sort.
//
// Kept tokens are a prefix of the tokens in descending order, and the drawn one is where the cumulated weights reach a target; so
// all that is asked of the order is where in it a count or a weight is reached. With z = l log2 e / T, tokens fall into bins of
// 1/32 octave of weight below an integer `ref` at or above the largest z; counts and sums of the bins give each border's bin, and only the members of
// those few bins are looked at one by one. Two kernels: the bins of pieces of rows; then a workgroup per row, which adds up the
// pieces' bins, collects the members of the bins that borders may fall into, and finds the borders among them.
//
// Weights are 2^(z - ref) to about 2^-52, as integers in steps of 2^-43: sums of integers do not depend on their order. (Weights in
// 32 bits would move the borders by about 2^-24 of the whole, and a border of 150000 flat weights comes every 2^-17.)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "internal.hpp"
#include "kserve.hpp"

namespace kcamd {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f32x4 f4a4 __attribute__((aligned(4)));
typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = 16, kBins = 1024, kList = 6144;
constexpr double kPerOctave = 32.0;
constexpr int kUnitBits = 43;  // (2^20 weights of up to 1 stay below 2^63)

struct SampleArgs {
    const float *logits, *u, *temperature, *top_p, *min_p;
    const int* top_k;
    int* tokens;
    float* probs;
    char* part;
    long long row;
    int rows, n, piece, pieces;
};

// A piece's bins in the workspace.
struct Piece {
    u64 sum[kBins];
    unsigned count[kBins];
    double ref;  // -infinity: no finite logit
    int wild;    // NaN or +infinity among the logits
    float top;   // the largest logit
};

// Octaves of weight per unit of logit. (Rows that take the likeliest token count as temperature 1.)
__device__ __forceinline__ bool greedy(float t) { return !(t > 0.0f); }
__device__ __forceinline__ double slopeOf(const SampleArgs& a, int r) {
    const float t = a.temperature ? a.temperature[r] : 1.0f;
    return greedy(t) ? 1.4426950408889634 : 1.4426950408889634 / (double)t;
}
// 2^x for x <= 0 in steps of 2^-43: the series of exp(r ln 2), |r| <= 1/2, whose 13th term is below 2^-52.
__device__ __forceinline__ u64 weightOf(double x) {
    if (x < -50.0) return 0;
    const double n = rint(x), r = (x - n) * 0.6931471805599453;
    double p = 1.0 / 479001600.0;
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const double scale = __builtin_bit_cast(double, (u64)(1023 + kUnitBits + (int)n) << 52);
    return (u64)fma(p, scale, 0.5);
}
// The bin below ref; the last one takes all that is further.
__device__ __forceinline__ int binOf(double z, double ref) {
    const double d = (ref - z) * kPerOctave;
    return d < kBins - 1 ? (int)d : kBins - 1;
}

// ---------------------------------------------------------------------------------------------- bins of the pieces
// 1024 threads hold a piece of 1024 R logits in registers: its maximum first, which gives ref, then the bins by atomics in LDS (the
// last one, into which all of a peaked row's tail falls, in registers).
template <int R>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(SampleArgs a) {
    __shared__ u64 sum[kBins];
    __shared__ unsigned count[kBins];
    __shared__ float tops[kWaves];
    __shared__ int wilds[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = blockIdx.y, p0 = blockIdx.x * a.piece, n = min(a.piece, a.n - p0);
    const float* x = a.logits + (long long)r * a.row + p0;
    const double c = slopeOf(a, r);
    f32x4 v[R / 4];
#pragma unroll
    for (int k = 0; k < R / 4; ++k) {
        const int at = 4 * (tid + kThreads * k);
        if (at + 3 < n) {
            v[k] = *reinterpret_cast<const f4a4*>(x + at);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[k][e] = at + e < n ? x[at + e] : -INFINITY;
        }
    }
    sum[tid] = 0;
    count[tid] = 0;
    float top = -INFINITY;
    bool wild = false;
#pragma unroll
    for (int k = 0; k < R / 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            wild |= !(v[k][e] < INFINITY);
            top = fmaxf(top, v[k][e]);
        }
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (lane == 0) tops[wave] = top;
    if (lane == 0) wilds[wave] = 0;
    if (__any(wild) && lane == 0) wilds[wave] = 1;
    __syncthreads();
    int any = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        top = fmaxf(top, tops[w]);
        any |= wilds[w];
    }
    Piece& out = reinterpret_cast<Piece*>(a.part)[(size_t)r * a.pieces + blockIdx.x];
    const bool empty = top == -INFINITY || any;
    const double ref = ceil((double)top * c);
    if (tid == 0) {
        out.ref = empty ? -INFINITY : ref;
        out.wild = any;
        out.top = top;
    }
    if (!empty) {
        u64 far = 0;
        unsigned farCount = 0;
#pragma unroll 4
        for (int k = 0; k < R / 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (v[k][e] == -INFINITY) continue;
                const double z = (double)v[k][e] * c;
                const int b = binOf(z, ref);
                const u64 w = weightOf(z - ref);
                if (b == kBins - 1) {
                    far += w;
                    ++farCount;
                } else {
                    atomicAdd(sum + b, w);
                    atomicAdd(count + b, 1u);
                }
            }
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            far += __shfl_xor(far, o);
            farCount += __shfl_xor(farCount, o);
        }
        if (lane == 0 && farCount) {
            atomicAdd(sum + kBins - 1, far);
            atomicAdd(count + kBins - 1, farCount);
        }
    }
    __syncthreads();
    out.sum[tid] = sum[tid];
    out.count[tid] = count[tid];
}

// ---------------------------------------------------------------------------------------------- borders and the draw
// Tokens in order: codes that ascend with (falling logit, rising number), unique.
__device__ __forceinline__ u64 codeOf(float l, int at) {
    const uint32_t u = __builtin_bit_cast(uint32_t, l == 0.0f ? 0.0f : l);
    const uint32_t up = u & 0x80000000u ? ~u : u | 0x80000000u;  // ascending with l
    return (u64)~up << 20 | (unsigned)at;
}
__device__ __forceinline__ float logitOf(u64 code) {
    const uint32_t up = ~(uint32_t)(code >> 20);
    return __builtin_bit_cast(float, up & 0x80000000u ? up & 0x7FFFFFFFu : ~up);
}

struct Shared {
    u64 sum[kBins];         // weights up to and with a bin
    unsigned count[kBins];  // tokens likewise
    u64 dsum[kBins];        // the digits of a search
    unsigned dcount[kBins];
    u64 list[kList];        // members of the wanted bins
    u64 few[64];
    u64 waves[kWaves], waves2[kWaves];
    u64 found[4];
    int bins[8];
    int listed, nfew;
};

__device__ __forceinline__ u64 waveScan(u64 x, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const u64 y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    return x;
}
// Sums up to and with this thread's of x and y.
__device__ __forceinline__ void scanTwo(u64& x, u64& y, u64* wx, u64* wy, int tid) {
    const int lane = tid & 63, wave = tid >> 6;
    x = waveScan(x, lane);
    y = waveScan(y, lane);
    __syncthreads();
    if (lane == 63) {
        wx[wave] = x;
        wy[wave] = y;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        x += w < wave ? wx[w] : 0;
        y += w < wave ? wy[w] : 0;
    }
}

__global__ __launch_bounds__(kThreads) void sample_draw_kernel(SampleArgs a) {
    extern __shared__ int4 lds4[];
    Shared& S = *reinterpret_cast<Shared*>(lds4);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x;
    const Piece* pieces = reinterpret_cast<const Piece*>(a.part) + (size_t)r * a.pieces;
    const float* x = a.logits + (long long)r * a.row;
    const double c = slopeOf(a, r);
    S.sum[tid] = 0;
    S.count[tid] = 0;
    if (tid == 0) S.listed = 0;
    double ref = -INFINITY;
    float top = -INFINITY;
    int wild = 0;
    for (int p = 0; p < a.pieces; ++p) {
        ref = fmax(ref, pieces[p].ref);
        top = fmaxf(top, pieces[p].top);
        wild |= pieces[p].wild;
    }
    if (wild || ref == -INFINITY) {
        if (tid == 0) {
            a.tokens[r] = -1;
            if (a.probs) a.probs[r] = 0.0f;
        }
        return;
    }
    __syncthreads();
    // bins of a piece lie (ref - its ref) octaves further
    auto shiftOf = [&](double pref) { return (int)fmin((ref - pref) * kPerOctave, (double)kBins); };
    for (int p = 0; p < a.pieces; ++p) {
        const double pref = pieces[p].ref;
        if (pref == -INFINITY) continue;
        const unsigned n = pieces[p].count[tid];
        if (!n) continue;
        const int down = (int)fmin(ref - pref, 63.0), to = min(kBins - 1, tid + shiftOf(pref));
        const u64 w = pieces[p].sum[tid];
        atomicAdd(S.sum + to, down ? ((w >> (down - 1)) + 1) >> 1 : w);
        atomicAdd(S.count + to, n);
    }
    __syncthreads();
    const u64 binSum = S.sum[tid], binCount = S.count[tid];
    u64 sumTo = binSum, countTo = binCount;
    scanTwo(sumTo, countTo, S.waves, S.waves2, tid);
    S.sum[tid] = sumTo;
    S.count[tid] = (unsigned)countTo;
    if (tid < 8) S.bins[tid] = kBins;
    __syncthreads();
    const unsigned finite = S.count[kBins - 1];
    auto sumBefore = [&](int b) { return b ? S.sum[b - 1] : 0ull; };
    // the first bin at which cond(sum, count up to it) holds, among all threads' bins; kBins if none
    auto firstBin = [&](int slot, bool here) {
        const unsigned long long v = __ballot(here);
        if (v && lane == 0) atomicMin(S.bins + slot, wave * 64 + __builtin_ctzll(v));
    };

    // ---- the cuts
    const float t = a.temperature ? a.temperature[r] : 1.0f;
    const float p = a.top_p ? a.top_p[r] : 1.0f, mp = a.min_p ? a.min_p[r] : 0.0f;
    const int tk = a.top_k ? a.top_k[r] : 0;
    unsigned K = tk > 0 ? min((unsigned)tk, finite) : finite;
    if (greedy(t) || p <= 0.0f || mp > 1.0f) K = 1;
    const bool cutP = p < 1.0f && K > 1, cutM = mp > 0.0f && K > 1;
    double u = a.u[r];
    u = u > 0.0 ? u : 0.0;
    // the largest token lies in the first bin that has one
    firstBin(0, S.count[tid] > 0);
    firstBin(1, S.count[tid] >= K);
    __syncthreads();
    const int b0 = S.bins[0], bK = S.bins[1];
    // what is kept of top_k: between kLo and kHi
    const bool cutK = K < S.count[bK];  // (else its bin is whole, and so is the sum)
    u64 kLo = cutK ? sumBefore(bK) : S.sum[bK], kHi = S.sum[bK];
    auto targetP = [&](u64 s) { return max((u64)ceil((double)p * (double)s), 1ull); };
    int bP0 = kBins, bP1 = kBins;
    if (cutP) {
        firstBin(2, S.sum[tid] >= targetP(kLo));
        firstBin(3, S.sum[tid] >= targetP(kHi));
    }
    __syncthreads();
    if (cutP) {
        bP0 = min(S.bins[2], bK);
        bP1 = min(S.bins[3], bK);
    }
    // min_p: where 2^(z - largest z) comes to it, a bin or so
    int bM0 = kBins, bM1 = kBins;
    if (cutM) {
        const double d = -log2((double)mp) * kPerOctave + b0;  // (bins below the largest token's upper end)
        bM0 = max(0, (int)fmin(d, 2000.0) - 1);
        bM1 = min(kBins - 1, bM0 + 3);
        bM0 = min(bM0, kBins - 1);
    }
    // the whole sum, and the draw's target: between these
    const int lo = min(min(bK, bP0), bM0), hi = min(min(bK, bP1), bM1);
    const u64 sLo = cutP || cutM ? sumBefore(lo) : kLo, sHi = cutP || cutM ? S.sum[hi] : kHi;
    auto targetU = [&](u64 s) { return s ? min((u64)((double)s * u), s - 1) : 0ull; };
    firstBin(4, S.sum[tid] > targetU(sLo));
    firstBin(5, S.sum[tid] > targetU(sHi));
    __syncthreads();
    const int bU0 = min(S.bins[4], hi), bU1 = min(S.bins[5], hi);

    // ---- the members of those bins
    const int from[4] = {cutK ? bK : kBins, bP0, bM0, bU0}, to[4] = {cutK ? bK : -1, cutP ? bP1 : -1, cutM ? min(bM1, kBins - 1) : -1, bU1};
    float least[4], most[4];  // logits of a range, a bin further on either side (of the last bin: all)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const bool none = to[k] < from[k];
        most[k] = none ? -INFINITY : (float)((ref - (from[k] - 1) / kPerOctave) / c);
        least[k] = none ? INFINITY : to[k] == kBins - 1 ? -INFINITY : (float)((ref - (to[k] + 2) / kPerOctave) / c);
        if (!none && !(most[k] > -INFINITY)) most[k] = INFINITY;  // (a slope of 0: all logits are in one bin)
        if (!none && !(least[k] < INFINITY)) least[k] = -INFINITY;
        if (!none) {  // (what rounding to 32 bits may take off)
            most[k] += fabsf(most[k]) * 2.4e-7f;
            least[k] -= fabsf(least[k]) * 2.4e-7f;
        }
    }
    auto wanted = [&](int b) {
        bool w = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) w |= b >= from[k] && b <= to[k];
        return w;
    };
    // f(code, bin) for every finite logit in a wanted bin
    auto overRow = [&](auto&& f) {
        for (int pc = 0; pc < a.pieces; ++pc) {
            const double pref = pieces[pc].ref;
            if (pref == -INFINITY) continue;
            const int shift = shiftOf(pref), p0 = pc * a.piece, n = min(a.piece, a.n - p0);
            auto one = [&](float l, int at) {
                bool maybe = false;
#pragma unroll
                for (int k = 0; k < 4; ++k) maybe |= l >= least[k] && l <= most[k];
                if (!maybe || l == -INFINITY) return;
                const int b = min(kBins - 1, binOf((double)l * c, pref) + shift);
                if (wanted(b)) f(codeOf(l, at), b);
            };
            for (int i = 4 * tid; i < n; i += 4 * kThreads) {
                if (i + 3 < n) {
                    const f32x4 v = *reinterpret_cast<const f4a4*>(x + p0 + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) one(v[e], p0 + i + e);
                } else {
                    for (int e = 0; e < n - i; ++e) one(x[p0 + i + e], p0 + i + e);
                }
            }
        }
    };
    overRow([&](u64 code, int b) {
        const int at = atomicAdd(&S.listed, 1);
        if (at < kList) S.list[at] = code | (u64)b << 52;
    });
    __syncthreads();
    const int listed = S.listed;
    constexpr u64 kCode = (1ull << 52) - 1;
    // (longer lists are not kept: the row is gone over again each time)
    auto overList = [&](auto&& f) {
        if (listed <= kList) {
            for (int i = tid; i < listed; i += kThreads) f(S.list[i] & kCode, (int)(S.list[i] >> 52));
        } else {
            overRow(f);
        }
    };
    auto unitsOf = [&](u64 code) { return weightOf((double)logitOf(code) * c - ref); };

    // Among the members of bin b, in order: the one at which the count reaches `want` (byCount), or the weights exceed `want`; found[0]: the
    // weights up to and with it, found[1] its code, found[2] its own weight. Where rounding leaves no such member: the last one with a weight.
    auto search = [&](int b, u64 want, bool byCount) {
        u64 lowest = 0, highest = kCode, before = 0;
        unsigned n = S.count[b] - (b ? S.count[b - 1] : 0), nBefore = 0;
        while (n > 64) {
            // the members' range, then the digits of ten bits from its top
            __syncthreads();
            if (tid == 0) {
                S.found[0] = ~0ull;
                S.found[1] = 0;
            }
            S.dsum[tid] = 0;
            S.dcount[tid] = 0;
            __syncthreads();
            u64 mn = ~0ull, mx = 0;
            overList([&](u64 code, int bb) {
                if (bb == b && code >= lowest && code <= highest) {
                    mn = min(mn, code);
                    mx = max(mx, code);
                }
            });
#pragma unroll
            for (int o = 32; o; o >>= 1) {
                mn = min(mn, (u64)__shfl_xor(mn, o));
                mx = max(mx, (u64)__shfl_xor(mx, o));
            }
            if (lane == 0) {
                atomicMin(S.found, mn);
                atomicMax(S.found + 1, mx);
            }
            __syncthreads();
            lowest = S.found[0];
            highest = S.found[1];
            const int bits = 64 - __builtin_clzll((highest - lowest) | 1), shift = max(0, bits - 10);
            overList([&](u64 code, int bb) {
                if (bb == b && code >= lowest && code <= highest) {
                    const int d = (int)((code - lowest) >> shift);
                    atomicAdd(S.dsum + d, unitsOf(code));
                    atomicAdd(S.dcount + d, 1u);
                }
            });
            __syncthreads();
            const u64 ds = S.dsum[tid], dc = S.dcount[tid];
            u64 w = ds, k = dc;
            scanTwo(w, k, S.waves, S.waves2, tid);
            // the first digit that reaches it; if none does, the last that has a weight (a member)
            const bool here = dc && (byCount ? nBefore + k >= want : before + w > want);
            if (tid < 8) S.bins[tid] = tid == 6 ? kBins : -1;
            __syncthreads();
            firstBin(6, here);
            if (ds || (byCount && dc)) atomicMax(S.bins + 7, tid);
            __syncthreads();
            const int digit = S.bins[6] < kBins ? S.bins[6] : max(S.bins[7], 0);
            if (tid == digit) {
                S.found[0] = w - ds;
                S.found[1] = k - dc;
                S.found[2] = dc;
            }
            __syncthreads();
            before += S.found[0];
            nBefore += (unsigned)S.found[1];
            n = (unsigned)S.found[2];
            lowest += (u64)digit << shift;
            highest = min(highest, lowest + (1ull << shift) - 1);
            if (n == 0) break;  // (a bin without weights: nothing is drawn from it)
        }
        __syncthreads();
        if (tid == 0) S.nfew = 0;
        __syncthreads();
        overList([&](u64 code, int bb) {
            if (bb == b && code >= lowest && code <= highest) {
                const int at = atomicAdd(&S.nfew, 1);
                if (at < 64) S.few[at] = code;
            }
        });
        __syncthreads();
        if (wave == 0) {
            const int m = min(S.nfew, 64);
            const u64 mine = lane < m ? S.few[lane] : ~0ull;
            const u64 w = lane < m ? unitsOf(mine) : 0;
            u64 upTo = before;
            unsigned rank = nBefore;
            for (int i = 0; i < m; ++i) {
                const u64 other = S.few[i], ow = __shfl(w, i);
                if (other <= mine) {
                    upTo += ow;
                    ++rank;
                }
            }
            const bool reached = lane < m && (byCount ? rank >= want : upTo > want);
            // the first that reaches it, or else the last with a weight
            u64 best = reached ? mine : ~0ull, last = lane < m && (w || byCount) ? mine : 0;
#pragma unroll
            for (int o = 32; o; o >>= 1) {
                best = min(best, (u64)__shfl_xor(best, o));
                last = max(last, (u64)__shfl_xor(last, o));
            }
            const u64 pick = best != ~0ull ? best : last;
            if (lane < m && mine == pick) {
                S.found[0] = upTo;
                S.found[1] = mine;
                S.found[2] = w;
            }
        }
        __syncthreads();
    };

    u64 kept = kLo;  // the sum of what is kept
    if (cutK) {
        search(bK, K - (bK ? S.count[bK - 1] : 0), true);
        kept = sumBefore(bK) + S.found[0];
        __syncthreads();
    }
    const u64 keptK = kept;
    if (cutP) {
        const u64 want = targetP(keptK);
        // (between bP0 and bP1)
        int b = bP0;
        while (b < bP1 && S.sum[b] < want) ++b;
        if (want > sumBefore(b)) {
            search(b, want - 1 - sumBefore(b), false);
            kept = min(kept, sumBefore(b) + S.found[0]);
        }
        __syncthreads();
    }
    if (cutM) {
        // what of bins bM0 .. bM1 comes up to min_p of the largest logit's weight
        __syncthreads();
        if (tid == 0) S.found[0] = 0;
        __syncthreads();
        const double zTop = (double)top * c, least2 = log2((double)mp);
        u64 w = 0;
        overList([&](u64 code, int b) {
            if (b >= bM0 && b <= bM1 && (double)logitOf(code) * c - zTop >= least2) w += unitsOf(code);
        });
#pragma unroll
        for (int o = 32; o; o >>= 1) w += __shfl_xor(w, o);
        if (lane == 0 && w) atomicAdd(S.found, w);
        __syncthreads();
        kept = min(kept, sumBefore(bM0) + S.found[0]);
        __syncthreads();
    }
    // ---- the draw
    const u64 want = targetU(kept);
    int b = bU0;
    while (b < bU1 && S.sum[b] <= want) ++b;
    search(b, want >= sumBefore(b) ? want - sumBefore(b) : 0, false);
    if (tid == 0) {
        a.tokens[r] = (int)(S.found[1] & 0xFFFFF);
        if (a.probs) a.probs[r] = (float)((double)S.found[2] / (double)kept);
    }
}

int piecesOf(int rows, int n, int* piece) {
    // pieces of 16384 logits until they fill the GPU twice, of 32768 beyond (a piece's bins are 12 KiB to write and read)
    const int64_t small = ((int64_t)n + 16383) / 16384;
    *piece = small * rows <= 512 ? 16384 : 32768;
    return (int)(((int64_t)n + *piece - 1) / *piece);
}

}  // namespace

size_t sampleRowsPartBytes(int rows, int n_vocab) {
    int piece;
    return size_t(rows) * piecesOf(rows, n_vocab, &piece) * sizeof(Piece);
}

int launchSampleRows(const kcSampleRowsArgs& a, hipStream_t s) {
    if (a.rows == 0) return 0;
    SampleArgs p{a.logits, a.u, a.temperature, a.top_p, a.min_p, a.top_k, a.tokens, a.probs, static_cast<char*>(a.part), a.row, a.rows, a.n_vocab, 0, 0};
    p.pieces = piecesOf(a.rows, a.n_vocab, &p.piece);
    static const int ok = fromHip(hipFuncSetAttribute(reinterpret_cast<const void*>(sample_draw_kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                      (int)sizeof(Shared)), "sample_rows: LDS size");
    if (ok) return ok;
    if (p.piece == 16384) hipLaunchKernelGGL(sample_bins_kernel<16>, dim3(p.pieces, a.rows), dim3(kThreads), 0, s, p);
    else hipLaunchKernelGGL(sample_bins_kernel<32>, dim3(p.pieces, a.rows), dim3(kThreads), 0, s, p);
    if (int e = fromHip(hipGetLastError(), "sample_rows (bins)")) return e;
    hipLaunchKernelGGL(sample_draw_kernel, dim3(a.rows), dim3(kThreads), sizeof(Shared), s, p);
    return fromHip(hipGetLastError(), "sample_rows");
}

}  // namespace kcamd
