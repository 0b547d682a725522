// ksample.hip -- sample_rows: temperature, top-k, top-p, min-p and the draw from given random numbers, without a sort.
//
// Kept tokens are a prefix of the tokens in descending order, and the drawn one is where the cumulated weights reach a target; so
// all that is asked of the order is where in it a count or a weight is reached. With z = l log2 e / T, tokens fall into bins of
// 1/32 octave of weight below an integer `ref` at or above the largest z; counts and weights of the bins give each border's bin, and only
// the members of those few bins are looked at one by one. Two kernels: the bins of pieces of rows; then a workgroup per row, which adds
// up the pieces' bins, collects the members of the bins that borders may fall into, and finds the borders among them.
//
// A weight is 2^-((b + 1/2) / 32), its bin's factor, times g = 2^-(s / 32) for the token's place s in the bin, |s| <= 1/2. A bin's sum of g
// is held as an integer in steps of 2^-38 (integers do not depend on the order of the atomics that add them up), with the
// count in the same word: one 64-bit atomic in LDS and a polynomial of degree 4 for each token. The bins' weights are added up
// in 64 bits, always in the same order. (Weights in 32 bits would move the borders by about 2^-24 of the whole, and among 150000 flat
// weights there is a border every 2^-17.)
//
// What bounds it: for many rows the bytes, which are read twice (512 rows of 151936: the bins 69 us, 4.5 TB/s, the draws 95 us, of which
// the second reading 55), for one row latencies, of one workgroup's steps one after the other (128256 logits, top_k 40: 5.5 and
// 15 us). A border among more members of its bins than the list holds costs readings of the row by one CU, two for each nine bits of
// the order: a row of 151936 under top_p 0.8 and temperatures of 0.5 to 1.5 takes 40 us where its logits' deviation is 2.5, 330 where it is
// 1, 780 where it is 0.3, 1570 where all are equal.
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
typedef u64 u64x2 __attribute__((ext_vector_type(2)));

// 64 octaves below ref in bins; the last bin takes what is further, less than 2^-62 of the largest weight: counted, but of weight 0
constexpr int kThreads = 1024, kWaves = 16, kDraw = 512, kBins = 2048, kFar = kBins - 1, kList = 5120, kGroups = 3 * kDraw, kPieces = 64;
constexpr double kPerOctave = 32.0;
constexpr int kUnitBits = 38;
constexpr u64 kUnit = 1ull << kUnitBits;

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
struct __attribute__((aligned(16))) Piece {
    u64 bins[kBins];  // sums of words: the count's multiple from bit 48 on, below it the sum of 2^38 (g - 1) + 2^32
    float top;        // the largest logit; -infinity: no finite one
    int wild;         // NaN or +infinity among the logits
    unsigned finite;  // finite logits
    float tops[kThreads];  // the largest of the logits that a thread held (4 each 4096)
};

// Four logits from number `at` on of the n at x; zeros from n on. (A load under a condition would be waited for before the next one.)
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rowOf(const float* x, int n) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(x), (short)0, __builtin_amdgcn_readfirstlane(4 * n), 0x00020000);
}
__device__ __forceinline__ f32x4 fourAt(__amdgpu_buffer_rsrc_t x, int at) {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(x, 4 * at, 0, 0));
}
// (Rows that take the likeliest token count as temperature 1.)
__device__ __forceinline__ bool greedy(float t) { return !(t > 0.0f); }
// A row's value of an array that may be null. (The load is unconditional, of u's in its place: under a condition each would be waited for.)
template <class T>
__device__ __forceinline__ T valueOf(const SampleArgs& a, const T* x, int r, T none) {
    const T y = (x ? x : reinterpret_cast<const T*>(a.u))[r];
    return x ? y : none;
}
// Octaves of weight per unit of logit.
__device__ __forceinline__ double slopeOf(const SampleArgs& a, int r) {
    const float t = valueOf(a, a.temperature, r, 1.0f);
    return greedy(t) ? 1.4426950408889634 : 1.4426950408889634 / (double)t;
}
// ref, and what the largest logit lies below it, in bins: within an octave, also where z is so large that integers are far apart.
__device__ __forceinline__ double refOf(float top, double slope) { return ceil((double)top * slope); }
__device__ __forceinline__ double offsetOf(float top, double slope, double ref) {
    return kPerOctave * fmin(fmax(fma(-(double)top, slope, ref), 0.0), 1.0);
}
// A token's distance below ref in bins (slope32 = 32 slope), its bin, and what it adds to the bin's word. g - 1 by the series of
// exp to the fourth power, the fifth's term (at most 2^-39.6) by the polynomial of degree 3 nearest to it (off by 2^-43.5); added to
// 2^14 + 2^10 + 1 / 64, so that the sum's last bit is 2^-38 and its bits but the last 33 are known.
__device__ __forceinline__ double distanceOf(float l, double top, double slope32, double offset) { return fma(top - (double)l, slope32, offset); }
__device__ __forceinline__ int binOf(double d) { return (int)fmin(d, (double)kFar); }
// The word's top 16 bits are the same for all, and odd: n words' sum gives n.
struct Series {
    double c[5];
};
__device__ __forceinline__ Series seriesOf() {
    constexpr double a = -0.6931471805599453 / kPerOctave, h2 = a * a / 4.0;  // (as)^5 ~ 5/4 h^2 (as)^3 - 5/16 h^4 as, |as| <= h
    Series r{{a * a * a * a / 24.0, a * a * a * (1.0 / 6.0 + 1.25 * h2 / 120.0), a * a / 2.0, a * (1.0 - 0.3125 * h2 * h2 / 120.0), 17408.0 + 1.0 / 64.0}};
    // (kept in registers, where the compiler would write them again for each token)
    asm("" : "+v"(r.c[0]), "+s"(r.c[1]), "+s"(r.c[2]), "+s"(r.c[3]), "+s"(r.c[4]));
    return r;
}
__device__ __forceinline__ u64 wordOf(const Series& k, double d) {
    const double s = __builtin_amdgcn_fract(d) - 0.5;
    return __builtin_bit_cast(u64, fma(fma(fma(fma(k.c[0], s, k.c[1]), s, k.c[2]), s, k.c[3]), s, k.c[4]));
}
constexpr unsigned kTop = 0x40D1, kTopInverse = 0x1831;  // of modulo 2^16
static_assert((kTop * kTopInverse & 0xFFFF) == 1);
__device__ __forceinline__ unsigned countOf(u64 words) { return (unsigned)(words >> 48) * kTopInverse & 0xFFFF; }
__device__ __forceinline__ u64 lowOf(u64 words) { return words & ((1ull << 48) - 1); }
// The sum of g of a bin of n tokens, from the sum of its words' low bits.
__device__ __forceinline__ u64 unitsOf(u64 words, unsigned n) { return words + (u64)n * (kUnit - (1ull << 32)); }
// The weight of a bin's unit.
constexpr int kOctave = 32;  // bins of an octave: of the factors of its bins (by octaves[], in LDS), which are computed once
__device__ __forceinline__ double factorOf(const double* octaves, int b) {
    return b < kFar ? ldexp(octaves[b % kOctave], -(b / kOctave) - kUnitBits) : 0.0;
}

// ---------------------------------------------------------------------------------------------- bins of the pieces
// 1024 threads hold a piece of 1024 R logits in registers: its maximum first, which gives ref, then the bins. (15 vector instructions a
// token, 40 us of the 69 above: what need not be is not done for each token.)
template <int R>
__global__ __launch_bounds__(kThreads, 8) void sample_bins_kernel(SampleArgs a) {
    __shared__ u64 bins[kBins];
    __shared__ float tops[kWaves];
    __shared__ unsigned wilds[kWaves], finites[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = blockIdx.y, p0 = blockIdx.x * a.piece, n = min(a.piece, a.n - p0);
    const float* x = a.logits + (long long)r * a.row + p0;
    const double slope = slopeOf(a, r);
    const auto row = rowOf(x, n);
    f32x4 v[R / 4];
#pragma unroll
    for (int k = 0; k < R / 4; ++k) v[k] = fourAt(row, 4 * (tid + kThreads * k));
    if (n < kThreads * R) {
#pragma unroll
        for (int k = 0; k < R / 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[k][e] = 4 * (tid + kThreads * k) + e < n ? v[k][e] : -INFINITY;
    }
    bins[tid] = 0;
    bins[tid + kThreads] = 0;
    float top = -INFINITY, odd = 0.0f;  // odd: NaN if some logit is not finite
    bool wild = false;
    unsigned finite = R;
#pragma unroll
    for (int k = 0; k < R / 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            odd = fmaf(v[k][e], 0.0f, odd);
            top = fmaxf(top, v[k][e]);
        }
    if (odd != 0.0f) {
        finite = 0;
#pragma unroll
        for (int k = 0; k < R / 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                wild |= !(v[k][e] < INFINITY);
                finite += v[k][e] > -INFINITY;
            }
    }
    Piece& out = reinterpret_cast<Piece*>(a.part)[(size_t)r * a.pieces + blockIdx.x];
    out.tops[tid] = top;
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        top = fmaxf(top, __shfl_xor(top, o));
        finite += __shfl_xor(finite, o);
    }
    const bool any = __any(wild);
    if (lane == 0) {
        tops[wave] = top;
        wilds[wave] = any;
        finites[wave] = finite;
    }
    __syncthreads();
    unsigned bad = 0;
    finite = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        top = fmaxf(top, tops[w]);
        bad |= wilds[w];
        finite += finites[w];
    }
    const bool empty = top == -INFINITY || bad;
    const Series series = seriesOf();
    const double top64 = top, slope32 = kPerOctave * slope, offset = offsetOf(top, slope, refOf(top, slope));
    if (!empty) {
#pragma unroll
        for (int k = 0; k < R / 4; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const double d = distanceOf(v[k][e], top64, slope32, offset);  // (infinite for a logit of -infinity; a slope of 0: NaN)
                if (d < kFar) atomicAdd(bins + (int)d, wordOf(series, d));  // (the others: those finite that no bin counts)
            }
    }
    __syncthreads();
    if (tid == 0) {
        out.top = top;
        out.wild = bad;
        out.finite = finite;
    }
    *reinterpret_cast<u64x2*>(out.bins + 2 * tid) = *reinterpret_cast<const u64x2*>(bins + 2 * tid);
}

// ---------------------------------------------------------------------------------------------- borders and the draw
// Tokens in order: codes of 52 bits that ascend with (falling logit, rising number).
__device__ __forceinline__ u64 codeOf(float l, int at) {
    const uint32_t u = __builtin_bit_cast(uint32_t, l == 0.0f ? 0.0f : l);
    const uint32_t up = u & 0x80000000u ? ~u : u | 0x80000000u;  // ascending with l
    return (u64)~up << 20 | (unsigned)at;
}
__device__ __forceinline__ float logitOf(u64 code) {
    const uint32_t up = ~(uint32_t)(code >> 20);
    return __builtin_bit_cast(float, up & 0x80000000u ? up & 0x7FFFFFFFu : ~up);
}
constexpr u64 kCode = (1ull << 52) - 1;

struct Shared {
    double sum[kBins];      // weights up to and with a bin
    unsigned count[kBins];  // tokens likewise
    union {
        unsigned groups[kGroups];
        struct {
            u64 dsum[kDraw];  // the digits of a search
            unsigned dcount[kDraw];
        };
    };
    u64 list[kList];        // members of the wanted bins, the bin from bit 52 on
    u64 few[64];
    double octaves[kOctave], top[kPieces], offset[kPieces];  // (64 pieces at most)
    int shift[kPieces];     // bins that a piece's lie further down
    u64 waves[kDraw / 64], waves2[kDraw / 64];
    u64 found[4], cut[4];
    float rowTop;
    int wild, bins[8], listed, grouped, nfew;
};
static_assert(sizeof(Shared) <= 80 * 1024);  // two workgroups on a CU

// Sums up to and with this thread's of x and y.
template <int Waves, class X, class Y>
__device__ __forceinline__ void scanTwo(X& x, Y& y, u64* wx, u64* wy, int tid) {
    const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const X p = __shfl_up(x, o);
        const Y q = __shfl_up(y, o);
        if (lane >= o) {
            x += p;
            y += q;
        }
    }
    __syncthreads();
    if (lane == 63) {
        reinterpret_cast<X*>(wx)[wave] = x;
        reinterpret_cast<Y*>(wy)[wave] = y;
    }
    __syncthreads();
    X xb = 0;
    Y yb = 0;
#pragma unroll
    for (int w = 0; w < Waves; ++w) {
        xb += w < wave ? reinterpret_cast<X*>(wx)[w] : 0;
        yb += w < wave ? reinterpret_cast<Y*>(wy)[w] : 0;
    }
    x += xb;
    y += yb;
}

// Lane i's value, i the same for all.
__device__ __forceinline__ u64 laneOf(u64 x, int i) {
    return (u64)(unsigned)__builtin_amdgcn_readlane((int)(x >> 32), i) << 32 | (unsigned)__builtin_amdgcn_readlane((int)x, i);
}
__device__ __forceinline__ int same(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float same(float x) { return __builtin_bit_cast(float, same(__builtin_bit_cast(int, x))); }
__device__ __forceinline__ double same(double x) {
    const u64 u = __builtin_bit_cast(u64, x);
    return __builtin_bit_cast(double, (u64)(unsigned)same((int)(u >> 32)) << 32 | (unsigned)same((int)u));
}

// (512 threads: two workgroups on a CU, one's reads beside the other's searches; 512 rows of 151936: 117 us, 130 with 1024. One row: the same.)
__global__ __launch_bounds__(kDraw, 4) void sample_draw_kernel(SampleArgs a) {
    extern __shared__ int4 lds4[];
    Shared& S = *reinterpret_cast<Shared*>(lds4);
    // (the last rows first: they were read last, and lie in the caches still)
    constexpr int NT = kDraw, BPT = kBins / NT, kDigitBits = 9;
    static_assert(1 << kDigitBits == NT);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = a.rows - 1 - blockIdx.x;
    const Piece* pieces = reinterpret_cast<const Piece*>(a.part) + (size_t)r * a.pieces;
    const float* x = a.logits + (long long)r * a.row;
    const double slope = slopeOf(a, r), slope32 = kPerOctave * slope;
    const float t = valueOf(a, a.temperature, r, 1.0f), p = valueOf(a, a.top_p, r, 1.0f), mp = valueOf(a, a.min_p, r, 0.0f);
    const int tk = valueOf(a, a.top_k, r, 0);
    double u = a.u[r];
    unsigned finite = 0;
    if (wave == 0) {
        const bool in = lane < a.pieces;
        const Piece& piece = pieces[min(lane, a.pieces - 1)];
        const float topHere = piece.top, mine = in ? topHere : -INFINITY;
        const int wildHere = piece.wild;
        const unsigned finiteHere = piece.finite;
        const bool wild = __any(in && wildHere);
        finite = in ? finiteHere : 0;
        float top = mine;
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            top = fmaxf(top, __shfl_xor(top, o));
            finite += __shfl_xor(finite, o);
        }
        const bool none = mine == -INFINITY;
        const double ref = refOf(mine, slope);
        S.top[lane] = mine;
        S.offset[lane] = offsetOf(mine, slope, ref);
        S.shift[lane] = none ? kBins : (int)fmin((refOf(top, slope) - ref) * kPerOctave, (double)kBins);
        if (lane == 0) {
            S.rowTop = top;
            S.wild = wild;
            S.found[0] = finite;
            S.listed = S.grouped = 0;
        }
    }
    float ahead[8][kThreads / NT];  // (of the first pieces: on the way while the bins are looked at)
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int h = 0; h < kThreads / NT; ++h) ahead[k][h] = pieces[min(k, a.pieces - 1)].tops[tid + NT * h];
    if (tid < 8) S.bins[tid] = kBins;
    if (wave == 1 && lane < kOctave) S.octaves[lane] = exp2(-(lane + 0.5) / kPerOctave);
    __syncthreads();
    if (S.wild || S.rowTop == -INFINITY) {
        if (tid == 0) {
            a.tokens[r] = -1;
            if (a.probs) a.probs[r] = 0.0f;
        }
        return;
    }
    const double top = same(S.rowTop);
    finite = same((int)S.found[0]);

    // ---- the row's bins: BPT a thread, of all pieces (their shifts are multiples of 32)
    unsigned cnt[BPT] = {};
    u64 words[BPT] = {};
    for (int p0 = 0; p0 < a.pieces; p0 += 8) {
        u64x2 y[8][BPT / 2];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int pc = min(p0 + k, a.pieces - 1), at = BPT * tid - S.shift[pc];
            const bool in = p0 + k < a.pieces && at >= 0;
#pragma unroll
            for (int e = 0; e < BPT / 2; ++e) {
                y[k][e] = *reinterpret_cast<const u64x2*>(pieces[pc].bins + max(at, 0) + 2 * e);
                if (!in) y[k][e] = u64x2{0, 0};
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < BPT; ++e) {
                cnt[e] += countOf(y[k][e / 2][e % 2]);
                words[e] += lowOf(y[k][e / 2][e % 2]);
            }
    }
    if (tid == NT - 1) cnt[BPT - 1] = words[BPT - 1] = 0;  // (the last bin)
    double sumTo[BPT], own = 0.0;  // weights up to and with a bin, tokens likewise
    unsigned countTo[BPT], n = 0;
#pragma unroll
    for (int e = 0; e < BPT; ++e) {
        own += factorOf(S.octaves, BPT * tid + e) * (double)unitsOf(words[e], cnt[e]);
        sumTo[e] = own;
        n += cnt[e];
        countTo[e] = n;
    }
    // Sums by halves: to those of a right half its left half's last one is added. So, roundings included, none is below the bin's before
    // it and none differs from it where the bin has no token: what a comparison of sums finds is a bin with tokens, and u times a sum
    // is reached below it. (Where each sum was added up in its own way, an empty bin's could lie a rounding above the last one with tokens,
    // and a number of 1 or more draw from there.)
    unsigned upTo = n;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const unsigned k = __shfl_up(upTo, o);
        const double left = __shfl(sumTo[BPT - 1], (lane & -2 * o) + o - 1);
        if (lane >= o) upTo += k;
        if (lane & o) {
#pragma unroll
            for (int e = 0; e < BPT; ++e) sumTo[e] += left;
        }
    }
    if (lane == 63) {
        reinterpret_cast<double*>(S.waves)[wave] = sumTo[BPT - 1];
        S.waves2[wave] = upTo;
    }
    __syncthreads();
    {
        double left = 0.0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) {
            left += w < wave ? reinterpret_cast<const double*>(S.waves)[w] : 0.0;
            upTo += w < wave ? (unsigned)S.waves2[w] : 0u;
        }
#pragma unroll
        for (int e = 0; e < BPT; ++e) S.sum[BPT * tid + e] = sumTo[e] = left + sumTo[e];
    }
    if (tid == NT - 1) {
        cnt[BPT - 1] = finite - upTo;
        countTo[BPT - 1] = finite - (upTo - n);
    }
#pragma unroll
    for (int e = 0; e < BPT; ++e) {
        countTo[e] += upTo - n;
        S.count[BPT * tid + e] = countTo[e];
    }
    auto sumBefore = [&](int b) { return b ? S.sum[b - 1] : 0.0; };
    auto countBefore = [&](int b) { return b ? S.count[b - 1] : 0u; };
    // the first bin with a token at which cond(its number among the thread's) holds, kBins if none; to S.bins[slot]
    auto firstBin = [&](int slot, auto&& cond) {
        int first = kBins;
#pragma unroll
        for (int e = BPT - 1; e >= 0; --e) first = cnt[e] && cond(e) ? BPT * tid + e : first;
        const unsigned long long v = __ballot(first < kBins);
        if (v && lane == __builtin_ctzll(v)) atomicMin(S.bins + slot, first);
    };

    // ---- the cuts
    unsigned K = tk > 0 ? min((unsigned)tk, finite) : finite;
    if (greedy(t) || p <= 0.0f || mp > 1.0f) K = 1;
    bool cutP = p < 1.0f && K > 1, cutM = mp > 0.0f && K > 1;
    u = u > 0.0 ? fmin(u, 0x1.fffffffffffffp-1) : 0.0;
    firstBin(0, [&](int) { return true; });  // the largest token's
    firstBin(1, [&](int e) { return countTo[e] >= K; });
    __syncthreads();
    const int b0 = same(S.bins[0]), bK = same(S.bins[1]);
    // what top_k keeps: between kLo and kHi
    const bool cutK = K < S.count[bK] && bK < kFar;  // (else its bin is whole, or of no weight)
    const double kHi = S.sum[bK], kLo = cutK ? sumBefore(bK) : kHi;
    int bP0 = kBins, bP1 = kBins;
    if (cutP) {
        firstBin(2, [&](int e) { return sumTo[e] >= p * kLo; });
        firstBin(3, [&](int e) { return sumTo[e] >= p * kHi; });
    }
    __syncthreads();
    if (cutP) {
        bP0 = min(same(S.bins[2]), bK);
        bP1 = min(same(S.bins[3]), bK);
    }
    // min_p: where 2^(z - largest z) comes to it, a bin or so
    int bM0 = kBins, bM1 = kBins;
    if (cutM) {
        const double d = b0 - log2((double)mp) * kPerOctave;  // (bins below the upper end of the largest token's)
        cutM = d < kFar - 4;                                  // (else it cuts off nothing that has a weight)
        if (cutM) {
            bM0 = max(0, (int)d - 1);
            bM1 = bM0 + 3;
        }
        if (cutM && cutP && bM1 < bP0) {  // (top_p cuts further down: it does not matter)
            cutP = false;
            bP0 = bP1 = kBins;
        } else if (cutM && cutP && bP1 < bM0) {
            cutM = false;
            bM0 = bM1 = kBins;
        }
    }
    // the whole sum, and the draw's target: between these
    const int lo = min(min(bK, bP0), bM0), hi = min(min(bK, bP1), bM1);
    const double sLo = cutP || cutM ? sumBefore(lo) : kLo, sHi = cutP || cutM ? S.sum[hi] : kHi;
    firstBin(4, [&](int e) { return sumTo[e] > u * sLo; });
    firstBin(5, [&](int e) { return sumTo[e] > u * sHi; });
    __syncthreads();
    const int bU0 = min(same(S.bins[4]), hi), bU1 = min(same(S.bins[5]), hi);

    // ---- the members of those bins: of the draw's, the cuts' by weight (which overlap where there are two), the cut's by count
    const int from[3] = {bU0, min(bP0, bM0), cutK ? bK : kBins};
    const int to[3] = {bU1, max(cutP ? bP1 : -1, cutM ? bM1 : -1), cutK ? bK : -1};
    const double offset = offsetOf(same(S.rowTop), slope, refOf(same(S.rowTop), slope));
    // Their logits, and what rounding may take off: |l - mid| - half below 0 for one of them.
    const double perBin = 1.0 / slope32;
    float mid[3], half[3], lowest = INFINITY;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        constexpr float kMost = 3.402823466e38f;  // (nothing here may be infinite: the difference of two is NaN, which is nobody's neighbour)
        const float hiL = (float)fmax(fmin(top - (from[k] - offset) * perBin, (double)kMost), -(double)kMost);
        const float loL = (float)fmax(fmin(top - (to[k] + 1 - offset) * perBin, (double)kMost), -(double)kMost);
        const float slack = 2.4e-7f * fmaxf((float)fabs(top), 1.2e-38f);
        const bool none = to[k] < from[k], all = slope == 0.0;  // (a slope of 0: all logits lie in one bin)
        const float hi = fminf(fmaf(fabsf(hiL), 2.4e-7f, hiL) + slack, kMost), lo = fmaxf(fminf(fmaf(fabsf(loL), -2.4e-7f, loL) - slack, 3.4e38f), -kMost);
        const float m = 0.5f * lo + 0.5f * hi;
        mid[k] = same(none || all ? 0.0f : m);
        half[k] = same(none ? -INFINITY : all ? INFINITY : fmaxf(hi - m, m - lo) * 1.000001f + 1.2e-38f);
        lowest = fminf(lowest, same(none ? INFINITY : all ? -INFINITY : lo));
    }
    auto near = [&](float l) {  // (its sign bit)
        const float x0 = fabsf(l - mid[0]) - half[0], x1 = fabsf(l - mid[1]) - half[1], x2 = fabsf(l - mid[2]) - half[2];
        return __builtin_bit_cast(unsigned, fminf(fminf(x0, x1), x2));
    };
    auto binAt = [&](float l, int at) {
        const int pc = at / a.piece;
        return min(binOf(distanceOf(l, S.top[pc], slope32, S.offset[pc])) + S.shift[pc], kFar);
    };
    // Of 4 K values, at at0 + step k, those of the members. (They are few, and read again: which register holds one is not known in
    // advance.)
    const auto row = rowOf(x, a.n);
    auto keep = [&](auto&& v, int at0, int step) {
        constexpr int K = sizeof v / sizeof v[0];
        unsigned mask = 0;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) mask = __builtin_amdgcn_alignbit(mask, near(v[k][e]), 31);  // (the first one's bit on top)
        if (at0 + step * (K - 1) + 3 >= a.n)
            for (int i = 0; i < 4 * K; ++i)
                if (at0 + step * (i >> 2) + (i & 3) >= a.n) mask &= ~(1u << (4 * K - 1 - i));
        if (!mask) return;
        int pos = atomicAdd(&S.listed, __builtin_popcount(mask));
        for (; mask; mask &= mask - 1, ++pos) {
            const int i = 4 * K - 1 - __builtin_ctz(mask), at = at0 + step * (i >> 2) + (i & 3);
            if (pos < kList) S.list[pos] = codeOf(x[at], at);
        }
    };
    // The groups whose largest logit is not below all of them: few where the borders are among a row's first tokens (one row of 128256
    // with top_k 40: 4.5 us, 14 for all logits). Of more than there is room for all logits are read.
    for (int p0 = 0; p0 < a.pieces; p0 += 8) {
#pragma unroll
        for (int h = 0; h < kThreads / NT; ++h) {
            float tops[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) tops[k] = p0 ? pieces[min(p0 + k, a.pieces - 1)].tops[tid + NT * h] : ahead[k][h];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (p0 + k < a.pieces && tops[k] >= lowest) {
                    const int at = atomicAdd(&S.grouped, 1);
                    if (at < kGroups) S.groups[at] = (p0 + k) * a.piece + 4 * (tid + NT * h);
                }
        }
    }
    __syncthreads();
    const int grouped = same(S.grouped);
    if (grouped <= kGroups) {
        const int per = a.piece / (4 * kThreads), lgPer = per == 8 ? 3 : 2;
        for (int c0 = tid; c0 < grouped << lgPer; c0 += 2 * NT) {
            f32x4 v[2][1];
            int at[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int c = c0 + NT * k;
                at[k] = c < grouped << lgPer ? (int)S.groups[c >> lgPer] + 4 * kThreads * (c & (per - 1)) : a.n;
                v[k][0] = fourAt(row, at[k]);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) keep(v[k], at[k], 0);
        }
    } else {
        // (the next ones are under way while these are looked at)
        constexpr int Step = 4 * NT;
        f32x4 v[4], w[4];
        auto load = [&](f32x4 (&z)[4], int i0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) z[k] = fourAt(row, i0 + Step * k);
        };
        load(v, 4 * tid);
        for (int i0 = 4 * tid; i0 < a.n; i0 += 8 * Step) {
            load(w, i0 + 4 * Step);
            keep(v, i0, Step);
            load(v, i0 + 8 * Step);
            keep(w, i0 + 4 * Step, Step);
        }
    }
    __syncthreads();
    const int listed = same(S.listed);
    // (no more than a wavefront has lanes: the first one does the rest by itself; the barriers do not wait for the others, which have ended)
    if (listed <= 64 && wave) return;
    if (listed <= kList) {
        for (int i = tid; i < listed; i += NT) {
            const u64 code = S.list[i];
            S.list[i] = code | (u64)binAt(logitOf(code), (int)(code & 0xFFFFF)) << 52;
        }
    }
    __syncthreads();
    // f(code, bin) for the members of the wanted bins (and some others). A list that is too long is not kept: the row is gone over
    // again each time.
    auto overList = [&](auto&& f) {
        const bool kept = listed <= kList;
        const int n = kept ? listed : a.n;
#pragma unroll 1
        for (int i = tid; i < n; i += NT) {
            u64 e;
            if (kept) {
                e = S.list[i];
            } else {
                const float l = x[i];
                if (!(near(l) >> 31) || l == -INFINITY) continue;
                e = codeOf(l, i) | (u64)binAt(l, i) << 52;
            }
            f(e & kCode, (int)(e >> 52));
        }
    };
    // a token's part of its bin's sum: what the first kernel added for it
    const Series series = seriesOf();
    auto unitOf = [&](u64 code) {
        const int pc = (int)(code & 0xFFFFF) / a.piece;
        return unitsOf(lowOf(wordOf(series, distanceOf(logitOf(code), S.top[pc], slope32, S.offset[pc]))), 1);
    };

    // Among the members of bin b, in order, the one with which the count (byCount) or the sum reaches `want`, the last one if none does:
    // found[0]: the sum up to and with it, found[1] its code, found[2] its own part.
    auto search = [&](int b, u64 want, bool byCount) {
        u64 lowest = 0, highest = kCode, before = 0;
        unsigned n = S.count[b] - countBefore(b), nBefore = 0;
        // (nine bits of a code of 52 each time, which are all different: six times at most)
        for (int round = 0; n > 64 && round < 6; ++round) {
            // the members' range, then the digits from its top
            __syncthreads();
            if (tid == 0) {
                S.found[0] = ~0ull;
                S.found[1] = 0;
                S.bins[6] = kBins;
                S.bins[7] = -1;
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
            if (lowest > highest) break;
            const int shift = max(0, 64 - __builtin_clzll((highest - lowest) | 1) - kDigitBits);
            overList([&](u64 code, int bb) {
                if (bb == b && code >= lowest && code <= highest) {
                    const int d = (int)((code - lowest) >> shift);
                    atomicAdd(S.dsum + d, unitOf(code));
                    atomicAdd(S.dcount + d, 1u);
                }
            });
            __syncthreads();
            const u64 ds = S.dsum[tid];
            const unsigned dc = S.dcount[tid];
            u64 w = ds;
            unsigned k = dc;
            scanTwo<NT / 64>(w, k, S.waves, S.waves2, tid);
            const unsigned long long here = __ballot(dc && (byCount ? nBefore + k >= want : before + w >= want)), some = __ballot(dc != 0);
            if (here && lane == 0) atomicMin(S.bins + 6, wave * 64 + __builtin_ctzll(here));
            if (some && lane == 0) atomicMax(S.bins + 7, wave * 64 + 63 - __builtin_clzll(some));
            __syncthreads();
            const int digit = S.bins[6] < kBins ? S.bins[6] : S.bins[7];
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
            const int m = min(same(S.nfew), 64);
            const u64 mine = lane < m ? S.few[lane] : ~0ull;
            const u64 w = lane < m ? unitOf(mine) : 0;
            u64 upTo = before;
            unsigned rank = 0;  // with itself
            for (int i = 0; i < m; ++i) {
                const u64 other = laneOf(mine, i), ow = laneOf(w, i);
                upTo += other <= mine ? ow : 0;
                rank += other <= mine;
            }
            // (the ones that do not reach it come first)
            const bool reached = byCount ? nBefore + rank >= want : upTo >= want;
            const int first = min(__builtin_popcountll(__ballot(lane < m && !reached)), m - 1);
            if (lane < m && (int)rank == first + 1) {
                S.found[0] = upTo;
                S.found[1] = mine;
                S.found[2] = w;
            }
        }
        __syncthreads();
    };
    // the first bin from b on, up to last, with a token and cond; else the last with a token
    auto walk = [&](int b, int last, auto&& cond) {
        while (b < last && !(S.count[b] > countBefore(b) && cond(b))) ++b;
        while (b > 0 && S.count[b] == countBefore(b)) --b;
        return b;
    };
    auto unitsTo = [&](int b, double target) { return fmax(0.0, fmin((target - sumBefore(b)) / factorOf(S.octaves, b), 0x1p60)); };

    double kept = kLo;  // the weight of what is kept
    // Where what is kept ends: its last bin, and what of that bin is kept. The draw's target is below the kept weight, but for roundings:
    // it is looked for no further than here.
    int lastBin = kBins;
    u64 lastUnits = 0;
    auto keepTo = [&](int b, u64 units) {
        if (b < lastBin || (b == lastBin && units < lastUnits)) {
            lastBin = b;
            lastUnits = units;
        }
    };
    for (int stage = 0; stage < 3; ++stage) {  // the cuts by count and by weight, the draw
        int b = bK;
        u64 want;
        if (stage == 0) {
            if (!cutK) continue;
            want = K - countBefore(bK);
        } else if (stage == 1) {
            if (!cutP) continue;
            const double target = p * kept;
            b = walk(bP0, bP1, [&](int k) { return S.sum[k] >= target; });
            want = max((u64)ceil(unitsTo(b, target)), 1ull);
        } else {
            if (cutM) {  // what of bins bM0 .. bM1 comes up to min_p of the largest logit's weight
                __syncthreads();
                if (tid < 4) S.cut[tid] = 0;
                __syncthreads();
                const double least2 = log2((double)mp);
                overList([&](u64 code, int bb) {
                    if (bb >= bM0 && bb <= bM1 && ((double)logitOf(code) - top) * slope >= least2) atomicAdd(S.cut + (bb - bM0), unitOf(code));
                });
                __syncthreads();
                double s = sumBefore(bM0);
#pragma unroll
                for (int k = 0; k < 4; ++k) s += factorOf(S.octaves, bM0 + k) * (double)S.cut[k];
                kept = fmin(kept, s);
                int k = 3;
                while (k >= 0 && !S.cut[k]) --k;
                if (k >= 0) keepTo(bM0 + k, S.cut[k]);
                else keepTo(bM0 - 1, ~0ull);
            }
            const double target = u * kept;
            b = walk(bU0, min(bU1, lastBin), [&](int k) { return S.sum[k] > target; });
            want = (u64)unitsTo(b, target) + 1;
            if (b == lastBin) want = min(want, lastUnits);
        }
        b = same(b);
        search(b, want, stage == 0);
        if (stage == 2) {
            if (tid == 0) {
                a.tokens[r] = (int)(S.found[1] & 0xFFFFF);
                if (a.probs) a.probs[r] = (float)(factorOf(S.octaves, b) * (double)S.found[2] / kept);
            }
        } else {
            const double s = sumBefore(b) + factorOf(S.octaves, b) * (double)S.found[0];
            kept = stage == 0 ? s : fmin(kept, s);
            keepTo(b, S.found[0]);
            __syncthreads();
        }
    }
}

int piecesOf(int rows, int n, int* piece) {
    // Pieces of 32768 logits, which are 16 KiB of bins each to write and read; of 16384 for few rows, which then have more workgroups, and for small
    // vocabularies, which would be one piece or two. (us with pieces of 16384 / 32768: 128256 logits, 1 row 22.3 / 25.4; 151936 logits, 8 rows
    // 26.1 / 26.0, 32 rows 36.8 / 33.2, 256 rows 66.3 / 62.8; 32000 logits, 1 row 21.5 / 22.7, 64 rows 24.2 / 26.7, 256 rows 32.7 / 33.9.)
    const int small = (n + 16383) / 16384;
    *piece = n <= 65536 || (int64_t)small * rows <= 64 ? 16384 : 32768;
    return (n + *piece - 1) / *piece;
}

}  // namespace

size_t sampleRowsPartBytes(int rows, int n_vocab) {
    // (fewer rows may have more pieces: what is enough for some is enough for fewer)
    int piece;
    const int small = (n_vocab + 16383) / 16384, few = std::min(rows, 64 / small);
    return std::max(size_t(rows) * piecesOf(rows, n_vocab, &piece), size_t(few) * piecesOf(few, n_vocab, &piece)) * sizeof(Piece);
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
    hipLaunchKernelGGL(sample_draw_kernel, dim3(a.rows), dim3(kDraw), sizeof(Shared), s, p);
    return fromHip(hipGetLastError(), "sample_rows");
}

}  // namespace kcamd
