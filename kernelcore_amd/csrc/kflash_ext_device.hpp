// kflash_ext_device.hpp -- what the attention kernels over a key/value cache share on the device: the packing of query rows, 4-bit
// blocks as matrix operands, score shaping.
//
// Query rows. The G = H / H_kv query heads of a KV head read the same keys, so token i and head g G + x
// make row r = i G + x of KV head g, and a matrix tile's columns are consecutive rows: a single token of a
// group of 4 and four tokens of one head fill a tile alike.
//
// Precision. q and out are f32. q is scaled by a power of two so that its largest value is in [2^7, 2^8)
// and split into fp16 parts hi = fp16(q), lo = fp16(q - hi): the products with fp16 keys are within about
// 2^-22 of f32 ones. The softmax's p is split the same way. A 4-bit block's codes - 8 are exact fp16
// integers; its scale d multiplies the f32 sum over the block's 32 values (K), or each value (V): d (c - 8) has 15
// bits, so it is an fp16 value and an exact fp16 rest (a third matrix chain instead of a rounded value).
#pragma once

#include <cfloat>
#include <climits>

#include "kflash_ext.hpp"

namespace kcamd {
namespace fx {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef int i2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
// loads and stores at the alignment the callers' strides leave
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef u4 u4a4 __attribute__((aligned(4)));
typedef u4 u4a2 __attribute__((aligned(2)));
typedef uint32_t u32a2 __attribute__((aligned(2)));
typedef f32x4 f4a4 __attribute__((aligned(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef f32x2 f2a4 __attribute__((aligned(4)));
struct __attribute__((packed, aligned(4))) int4a4 {
    int x, y, z, w;
    __device__ operator int4() const { return {x, y, z, w}; }
};
typedef __attribute__((address_space(3))) s4* LdsS4;
typedef __attribute__((address_space(3))) i2* LdsI2;

constexpr float kLog2e = 1.44269504088896f;
constexpr float kLn2 = 0.693147180559945f;
constexpr int kNoKey = INT_MAX;  // the position of a row past the cache's end or in an empty slot

// Constants kept in registers, where one instruction can mask and merge a word with them.
struct NibbleMagic {
    uint32_t low, high, base;
};
__device__ __forceinline__ NibbleMagic nibbleMagic() {
    NibbleMagic m{0x000F000Fu, 0x00F000F0u, 0x64006400u};
    asm("" : "+s"(m.low));
    asm("" : "+s"(m.high));
    asm("" : "+v"(m.base));
    return m;
}
// Eight codes - 8 of a word as fp16, in the order of nibbles 0, 4, 1, 5, 2, 6, 3, 7. A nibble at the foot of the significand of
// 1024 reads 1024 + code, one four bits up 1024 + 16 code: less 1032, or / 16 less 72 (both exact).
__device__ __forceinline__ h8 nibbles(uint32_t w, const NibbleMagic& k) {
    const h2 off = {(_Float16)-1032.0f, (_Float16)-1032.0f}, off16 = {(_Float16)-72.0f, (_Float16)-72.0f};
    const h2 by16 = {(_Float16)0.0625f, (_Float16)0.0625f};
    const uint32_t w8 = w >> 8;
    const h2 a = __builtin_bit_cast(h2, (w & k.low) | k.base) + off;
    const h2 b = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & k.high) | k.base), by16, off16);
    const h2 c = __builtin_bit_cast(h2, (w8 & k.low) | k.base) + off;
    const h2 d = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w8 & k.high) | k.base), by16, off16);
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The codes - 8 of a word's low (or, of w >> 4, high) nibbles as fp16, in the order of its bytes
__device__ __forceinline__ void byteCodes(uint32_t w, h2& a, h2& b) {
    const h2 off = {(_Float16)1032.0f, (_Float16)1032.0f};
    const uint32_t m = w & 0x0F0F0F0Fu;
    a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, m, 0x07010700u)) - off;
    b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, m, 0x07030702u)) - off;
}
// A V scale whose products with codes leave fp16's range (|d| > 8188), or an infinity or NaN: its block stays out of
// the matrix products.
__device__ __forceinline__ bool wildScale(uint32_t bits) { return (bits & 0x7FFFu) > 0x6FFFu; }
// Which of two fp16 values of a word is an infinity or NaN: bits 15 and 31.
__device__ __forceinline__ uint32_t wildHalves(uint32_t w) { return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }

// q values of one row as fp16 hi / lo parts of x 2^shift, with the scale's sign. 2^shift is a factor f and, for rows of numbers so
// small that f would overflow, 2^more.
struct QScale {
    float f;
    int more;
    float c;  // the factor that makes a sum of scaled products a score
};
__device__ __forceinline__ QScale qScale(float top, float scale) {
    const int shift = top > 0.0f && top < INFINITY ? 8 - __builtin_amdgcn_frexp_expf(top) : 0, first = min(shift, 126);
    // (a scale of 0 in q itself: times an infinite key it is NaN)
    return {scale == 0.0f ? 0.0f : ldexpf(scale < 0.0f ? -1.0f : 1.0f, first), shift - first, ldexpf(fabsf(scale), -shift)};
}
// Two numbers as fp16 parts hi + lo. (x - hi in one instruction each; x must not come straight from a matrix instruction.)
__device__ __forceinline__ void splitTwo(float x0, float x1, h2& hi, h2& lo) {
    hi = h2{(_Float16)x0, (_Float16)x1};
    const uint32_t hb = __builtin_bit_cast(uint32_t, hi);
    float r0, r1;
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(hb), "v"(x0));
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(hb), "v"(x1));
    lo = h2{(_Float16)r0, (_Float16)r1};
}
template <int N>
__device__ __forceinline__ void qSplit(const float (&x)[N], const QScale& s, h2 (&hi)[N / 2], h2 (&lo)[N / 2]) {
    float y[N];
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = x[e] * s.f;
    if (__builtin_expect(__any(s.more > 0), 0)) {
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = ldexpf(y[e], s.more);
    }
#pragma unroll
    for (int e = 0; e < N; e += 2) splitTwo(y[e], y[e + 1], hi[e / 2], lo[e / 2]);
}

__device__ __forceinline__ void qSplit8(const float (&x)[8], const QScale& s, h8& hi, h8& lo) {
    h2 h[4], l[4];
    qSplit<8>(x, s, h, l);
    hi = h8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
    lo = h8{l[0][0], l[0][1], l[1][0], l[1][1], l[2][0], l[2][1], l[3][0], l[3][1]};
}

// What a query row brings to its scores.
struct Row {
    int token, head;
    bool live;
    int limit;  // the last position it sees (causal), prefix included
    int pos, doc;
    float slope;
};
__device__ __forceinline__ int limitOf(const FxParams& a, int pos) {
    return a.causal ? min(max(pos, a.prefix - 1), INT_MAX - 1) : INT_MAX - 1;
}
__device__ __forceinline__ Row rowOf(const FxParams& a, int kvh, int r) {
    Row w;
    w.live = r < a.rows;
    const int rr = w.live ? r : a.rows - 1;
    w.token = rr / a.G;
    w.head = kvh * a.G + (rr - w.token * a.G);
    w.pos = a.qpos ? a.qpos[w.token] : a.pos0 + w.token;
    w.limit = limitOf(a, w.pos);
    w.doc = a.qdoc ? a.qdoc[w.token] : 0;
    w.slope = a.slopes ? a.slopes[w.head] : 0.0f;
    return w;
}

// Scores in base 2: x = y log2 e. What shapes them, made once per workgroup.
struct Shape {
    float inv_cap;   // 0: no cap
    float p5[6];     // cap log2 e times the coefficients of tanh(y) / y in y^2, |y| <= 3/4
    float p[5], q[4];  // of the quotient for |y| <= 9, P times cap log2 e
    bool bias;
};
__device__ __forceinline__ float uniform(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
__device__ __forceinline__ Shape shapeOf(const FxParams& a) {
    Shape s{};
    s.bias = a.slopes != nullptr;
    if (a.softcap > 0.0f) {
        s.inv_cap = uniform(1.0f / a.softcap);
        const float k = uniform(a.softcap * kLog2e);
        const float p5[6] = {1.0f, -0.33332958817481995f, 0.1332540661096573f, -0.05334447696805f, 0.01958298869431019f, -0.0047163087874650955f};
        const float p[5] = {1.0f, 0.13381023705005646f, 0.003495586570352316f, 2.0609057173714973e-05f, 1.335463029050743e-08f};
        const float q[4] = {0.46714338660240173f, 0.025876976549625397f, 0.00032856324105523527f, 7.776545203341811e-07f};
#pragma unroll
        for (int i = 0; i < 6; ++i) s.p5[i] = uniform(k * p5[i]);
#pragma unroll
        for (int i = 0; i < 5; ++i) s.p[i] = uniform(k * p[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) s.q[i] = q[i];
    }
    return s;
}
// A row's k below, finite: a sum of 0 stays a score of 0 beside the smallest caps and the largest q.
__device__ __forceinline__ float capFactor(float c, const Shape& s) { return fminf(c * s.inv_cap, FLT_MAX); }
// x[v] = cap log2 e tanh(x[v] k), k = score factor / cap. Two relative minimax fits of tanh(y) / y in y^2: a polynomial for |y| <= 3/4
// (3e-8) and above that a quotient for |y| <= 9 (2e-8; beyond, tanh is 1 within 3e-8). A score's own size decides between them, so
// that no other key or query reaches its bits (one form for a wavefront, by its largest score, would let them); the quotient is
// branched around where no lane has use for it (mostly: caps lie well above the scores. 2048 tokens, 24 heads, cap 30: 89 us; cap
// 4, where a score in 400 takes it: 100). A form through exp would lose the small arguments' last bits. NaN stays NaN.
__device__ __forceinline__ float smallTanh(float y, const Shape& s) {  // over y
    const float u = y * y;
    float r = fmaf(u, s.p5[5], s.p5[4]);
#pragma unroll
    for (int i = 3; i >= 0; --i) r = fmaf(u, r, s.p5[i]);
    return r;
}
__device__ __forceinline__ float largeTanh(float x, const Shape& s) {
    const float y = __builtin_elementwise_maximum(__builtin_elementwise_minimum(x, 9.0f), -9.0f);
    const float u = y * y;
    float p = fmaf(u, s.p[4], s.p[3]), q = fmaf(u, s.q[3], s.q[2]);
    p = fmaf(u, p, s.p[2]);
    q = fmaf(u, q, s.q[1]);
    p = fmaf(u, p, s.p[1]);
    q = fmaf(u, q, s.q[0]);
    p = fmaf(u, p, s.p[0]);
    q = fmaf(u, q, 1.0f);
    return y * p * __builtin_amdgcn_rcpf(q);
}
template <int N>
__device__ __forceinline__ void capScores(float (&x)[N], float k, const Shape& s) {
    float top = 0.0f;
#pragma unroll
    for (int v = 0; v < N; ++v) {
        x[v] *= k;
        top = fmaxf(top, fabsf(x[v]));
    }
    if (!__any(top > 0.75f)) {
#pragma unroll
        for (int v = 0; v < N; ++v) {
            x[v] *= smallTanh(x[v], s);
            if (v % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (four at a time are enough to fill the unit; all at once take registers)
        }
        return;
    }
#pragma unroll
    for (int v = 0; v < N; ++v) {
        float r = x[v] * smallTanh(x[v], s);
        if (!(fabsf(x[v]) <= 0.75f)) r = largeTanh(x[v], s);
        x[v] = r;
        if (v % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
}

// exp2 on the transcendental unit: 0 below 2^-126, where the sums it joins do not see it
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// The factor of a row's sums that makes them base-2 scores (never 0: a masked sum is -infinity, and stays it).
__device__ __forceinline__ float factor2(float c) { return fmaxf(c * kLog2e, 1.17549435e-38f); }

// Maxima over the lanes 32 (16) apart, without LDS: a swap of one register's upper half (odd rows of 16) with a copy's lower half
// (even rows). (The results are copied before they are cast: a bit cast of a vector's element takes its first one.)
__device__ __forceinline__ float swap32Max(float x) {
    const int y = __builtin_bit_cast(int, x);
    const auto r = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    const int a = r[0], b = r[1];
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float swap16Max(float x) {
    const int y = __builtin_bit_cast(int, x);
    const auto r = __builtin_amdgcn_permlane16_swap(y, y, false, false);
    const int a = r[0], b = r[1];
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}

// N values (p 2^11) as fp16 parts hi + lo
template <int N>
__device__ __forceinline__ void splitParts(const float (&x)[N], h8 (&hi)[N / 8], h8 (&lo)[N / 8]) {
#pragma unroll
    for (int v = 0; v < N; v += 2) {
        h2 h, l;
        splitTwo(x[v], x[v + 1], h, l);
        hi[v >> 3][v & 7] = h[0];
        hi[v >> 3][(v & 7) + 1] = h[1];
        lo[v >> 3][v & 7] = l[0];
        lo[v >> 3][(v & 7) + 1] = l[1];
    }
}

// x[i] of registers for a lane's own i
template <int N>
__device__ __forceinline__ float pick(const float (&x)[N], int i) {
    float r = x[0];
#pragma unroll
    for (int e = 1; e < N; ++e) {
        r = i == e ? x[e] : r;
        asm("" : "+v"(r));  // (selects, not an indexed array, which would move x to memory)
    }
    return r;
}

// Over the wavefront, in registers: lanes ^ 1, ^ 2, mirrored in eight and 16, then rows and halves swapped.
template <int CTRL>
__device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xF, 0xF, false); }
template <int CTRL>
__device__ __forceinline__ float dppF(float v) { return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(int, v))); }
template <class T, class F>
__device__ __forceinline__ T waveAll(T x, F&& op) {
    auto with = [&](int y) { x = op(x, __builtin_bit_cast(T, y)); };
    with(dpp<0xB1>(__builtin_bit_cast(int, x)));
    with(dpp<0x4E>(__builtin_bit_cast(int, x)));
    with(dpp<0x141>(__builtin_bit_cast(int, x)));
    with(dpp<0x140>(__builtin_bit_cast(int, x)));
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), false, false);
    const int a = r[0], b = r[1];
    x = op(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
    const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x), false, false);
    const int c = s[0], d = s[1];
    return op(__builtin_bit_cast(T, c), __builtin_bit_cast(T, d));
}
__device__ __forceinline__ int waveMin(int x) {
    return __builtin_amdgcn_readfirstlane(waveAll(x, [](int a, int b) { return min(a, b); }));
}
__device__ __forceinline__ int waveMax(int x) {
    return __builtin_amdgcn_readfirstlane(waveAll(x, [](int a, int b) { return max(a, b); }));
}
__device__ __forceinline__ float halfBits(uint32_t b) { return (float)__builtin_bit_cast(_Float16, (unsigned short)b); }
__device__ __forceinline__ uint32_t loadHalf(const char* p) { return *reinterpret_cast<const unsigned short*>(p); }
__device__ __forceinline__ float waveMaxF(float x) {
    return waveAll(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float waveSumF(float x) {
    return waveAll(x, [](float a, float b) { return a + b; });
}

// The lanes' loads and stores of LDS before this are done before those after it (a wavefront's own LDS accesses run in
// order: only the compiler has to keep them so).
__device__ __forceinline__ void waveLds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ---- tiles of 32 keys x 32 rows (v_mfma_f32_32x32x16_f16; lane (j, h) = row j, lane half h)

// LDS bytes of a key's row as fp16: one pad chunk puts consecutive rows on different banks
template <int D>
constexpr int kKeyRow = 2 * D + 16;

// q of 32 rows, W values of each, on its way to operands: loaded with consecutive lanes on consecutive values (a lane half per
// row instead, as the operands have it, touches 32 cache lines an instruction and comes back to each four times: 4 us of a
// workgroup's start), divided into hi and lo there, and turned into operands (values 16 ks + 8 h .. + 8 of the lane's row)
// through LDS, as fp16.
template <int W>
struct RowQ {
    static constexpr int LPR = W / 4, RPI = 64 / LPR, N = 32 / RPI;  // lanes to a row, rows to an instruction, instructions
    f32x4 x[N];
    // at: where the q of row lane % 32 begins, in floats
    __device__ __forceinline__ void load(const float* q, long long at, int lane) {
        const int lo = (int)at, hi = (int)(at >> 32);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int src = n * RPI + lane / LPR;
            const long long o = (long long)(((unsigned long long)(unsigned)__shfl(hi, src) << 32) | (unsigned)__shfl(lo, src));
            x[n] = *reinterpret_cast<const f4a4*>(q + o + 4 * (lane % LPR));
        }
    }
    // the rows' largest magnitudes to top[row]
    __device__ __forceinline__ void tops(float* top, int lane) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float m = fmaxf(fmaxf(fabsf(x[n][0]), fabsf(x[n][1])), fmaxf(fabsf(x[n][2]), fabsf(x[n][3])));
            m = fmaxf(m, dppF<0xB1>(m));   // lane ^ 1
            m = fmaxf(m, dppF<0x4E>(m));   // ^ 2
            m = fmaxf(m, dppF<0x141>(m));  // the other four of eight
            if constexpr (LPR >= 16) m = fmaxf(m, dppF<0x140>(m));  // the other eight of 16
            if constexpr (LPR >= 32) m = swap16Max(m);
            if constexpr (LPR >= 64) m = swap32Max(m);
            if (lane % LPR == 0) top[n * RPI + lane / LPR] = m;
        }
    }
    // the hi parts of row r's values to rows of `stride` fp16, the lo parts to `low`; topOf(r): the row's largest magnitude
    template <class F>
    __device__ __forceinline__ void split(const FxParams& a, _Float16* hi, int stride, int lane, F&& topOf, h4 (&low)[N]) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int r = n * RPI + lane / LPR;
            const float y[4] = {x[n][0], x[n][1], x[n][2], x[n][3]};
            h2 u[2], w[2];
            qSplit<4>(y, qScale(topOf(r), a.scale), u, w);
            low[n] = h4{w[0][0], w[0][1], w[1][0], w[1][1]};
            *reinterpret_cast<h4*>(hi + r * stride + 4 * (lane % LPR)) = h4{u[0][0], u[0][1], u[1][0], u[1][1]};
        }
    }
    __device__ __forceinline__ void place(_Float16* to, int stride, int lane, const h4 (&v)[N]) const {
#pragma unroll
        for (int n = 0; n < N; ++n) *reinterpret_cast<h4*>(to + (n * RPI + lane / LPR) * stride + 4 * (lane % LPR)) = v[n];
    }
};

// The same for a wavefront alone (few rows, whose lines the lanes share): values 16 ks + 8 h .. + 8 of the lane's row, loaded first, divided
// into hi and lo when they are there; returns the factor of the row's scores.
template <int D>
__device__ __forceinline__ void loadRow32(const FxParams& a, const Row& row, int h, f32x4 (&x)[D / 8]) {
    const float* qp = a.q + (size_t)row.token * a.q_tok + (size_t)row.head * a.q_head + 8 * h;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) x[n] = *reinterpret_cast<const f4a4*>(qp + 16 * (n >> 1) + 4 * (n & 1));
}
template <int D>
__device__ __forceinline__ float splitRow32(const FxParams& a, const f32x4 (&x)[D / 8], h8 (&qh)[D / 16], h8 (&ql)[D / 16]) {
    float top = 0.0f;
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[n][e]));
    top = fmaxf(top, __shfl_xor(top, 32));
    const QScale qs = qScale(top, a.scale);
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[2 * ks + (e >> 2)][e & 3];
        qSplit8(y, qs, qh[ks], ql[ks]);
    }
    return qs.c;
}

// A block of 32 codes as four operands of 8 consecutive values.
__device__ __forceinline__ void blockCodes(const u4& raw, h8 (&code)[4]) {
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            h2 x, y;
            byteCodes(s ? raw[w] >> 4 : raw[w], x, y);
            h8& o = code[2 * s + (w >> 1)];
            o[4 * (w & 1)] = x[0];
            o[4 * (w & 1) + 1] = x[1];
            o[4 * (w & 1) + 2] = y[0];
            o[4 * (w & 1) + 3] = y[1];
        }
}

// Eight bytes of a block: the low codes and the high ones.
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void byteCodes8(const u2& raw, h8& lo, h8& hi) {
    h2 x[8];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        byteCodes(raw[w], x[2 * w], x[2 * w + 1]);
        byteCodes(raw[w] >> 4, x[4 + 2 * w], x[5 + 2 * w]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        lo[2 * e] = x[e][0];
        lo[2 * e + 1] = x[e][1];
        hi[2 * e] = x[4 + e][0];
        hi[2 * e + 1] = x[4 + e][1];
    }
}

// Where the fp16 scale of block b of key `key` of a tile lies in LDS: the 16 keys of a lane half in the order of its scores.
__device__ __forceinline__ int scaleAt(int b, int key) { return (2 * b + ((key >> 2) & 1)) * 16 + (key >> 3) * 4 + (key & 3); }

// Sums of scaled products of the lane's 16 keys, 8 (v / 4) + 4 h + v % 4, from key rows in LDS (fp16 values, or codes - 8
// and their blocks' scales as scaleAt places them: eight of them a read, each taken as fp16 by the multiply-add).
template <int D, bool Q4>
__device__ __forceinline__ void keyScores(const char* keys, const char* scales, int j, int h, const h8 (&qh)[D / 16],
                                          const h8 (&ql)[D / 16], float (&x)[16]) {
    f32x16 zero;
#pragma unroll
    for (int v = 0; v < 16; ++v) zero[v] = 0.0f;
    const char* kr = keys + j * kKeyRow<D> + 16 * h;
    if constexpr (Q4) {
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = 0.0f;
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
            const h8 k0 = *reinterpret_cast<const h8*>(kr + 64 * b), k1 = *reinterpret_cast<const h8*>(kr + 64 * b + 32);
            f32x16 s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, qh[2 * b], zero, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, qh[2 * b + 1], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, ql[2 * b], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, ql[2 * b + 1], s, 0, 0, 0);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const h8 d = *reinterpret_cast<const h8*>(scales + (2 * b + h) * 32 + 16 * g);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[8 * g + e] = fmaf((float)d[e], s[8 * g + e], x[8 * g + e]);
            }
        }
    } else {
        f32x16 s = zero;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const h8 ka = *reinterpret_cast<const h8*>(kr + 32 * ks);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qh[ks], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, ql[ks], s, 0, 0, 0);
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = s[v];
    }
}

// The mask's values of the lane's 16 keys of tile t (32 keys).
struct MaskWords {
    uint32_t w[8];
    __device__ __forceinline__ void load(const unsigned short* mrow, int t, int h, int T) {
        const int words = (T + 1) / 2;
        if ((t + 1) * 16 <= words) {  // (the same for the wavefront)
            const uint32_t* at = reinterpret_cast<const uint32_t*>(mrow) + t * 16 + 2 * h;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const u2 two = *reinterpret_cast<const __attribute__((aligned(4))) u2*>(at + 4 * g);
                w[2 * g] = two[0];
                w[2 * g + 1] = two[1];
            }
            return;
        }
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int at = t * 16 + 4 * g + 2 * h + e;
                w[2 * g + e] = at < words ? reinterpret_cast<const uint32_t*>(mrow)[at] : 0xFC00FC00u;
            }
    }
};

// (a masked place is -infinity whatever its key holds)
__device__ __forceinline__ float addMask(float x, uint32_t bits) {
    return bits == 0xFC00u ? -INFINITY : fmaf(halfBits(bits), kLog2e, x);
}

// Sums of products into shaped scores in base 2. c: the factor of the row's scores; kp: the keys' positions where they are not the
// tile's own (LDS, in groups of four at 8 g + 4 h), key0 the first of the lane's; mk the mask's values where there is one (a
// pointer to them, null without, would put them into memory).
__device__ __forceinline__ void shapeScores(float (&x)[16], float c, const Shape& shape, const Row& row, const int* kp, int key0,
                                            bool masked, const MaskWords& mk) {
    if (shape.inv_cap > 0.0f) {
        capScores(x, capFactor(c, shape), shape);
    } else {
        const float c2 = factor2(c);
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] *= c2;
    }
    if (shape.bias) {
        const float slope = -row.slope * kLog2e;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            int4 p = {key0 + 8 * g, key0 + 8 * g + 1, key0 + 8 * g + 2, key0 + 8 * g + 3};
            if (kp) p = *reinterpret_cast<const int4*>(kp + 8 * g);
            x[4 * g] = fmaf(slope, fabsf((float)(row.pos - p.x)), x[4 * g]);
            x[4 * g + 1] = fmaf(slope, fabsf((float)(row.pos - p.y)), x[4 * g + 1]);
            x[4 * g + 2] = fmaf(slope, fabsf((float)(row.pos - p.z)), x[4 * g + 2]);
            x[4 * g + 3] = fmaf(slope, fabsf((float)(row.pos - p.w)), x[4 * g + 3]);
        }
    }
    if (masked) {
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = addMask(x[v], (v & 1) ? mk.w[v >> 1] >> 16 : mk.w[v >> 1] & 0xFFFFu);
    }
}

// What the row does not see becomes -infinity: by the keys' positions and document numbers in LDS.
__device__ __forceinline__ void hideKeys(float (&x)[16], const Row& row, const int* kp, const int* kd) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int4 a = *reinterpret_cast<const int4*>(kp + 8 * g), b = *reinterpret_cast<const int4*>(kd + 8 * g);
        const int p[4] = {a.x, a.y, a.z, a.w}, d[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * g + e] = p[e] <= row.limit && d[e] == row.doc ? x[4 * g + e] : -INFINITY;
    }
}

// ---- keys and queries that hold an infinity or NaN
// On the matrix cores such a number makes a row's sum infinite or NaN, but NaN also where the definition says infinity: an infinite key meets
// a low part of q that is 0 or of the other sign. A sum that comes out infinite is right (of a 4-bit block, whose scale multiplies
// the sum of its products, an infinite scale is replaced by NaN: finiteOrNaN). So the kernels run on as they are, and a row
// (attn_weights: a position) whose sum of weights is NaN at the end is made again from the definition in plain f32 by a wavefront: at
// the first such score where it is NaN by definition too (1000 tokens of NaN over 1024 positions, 32 heads of 128: 0.2 ms), else
// slowly (every row to be made again: 2.4 ms; of one token over 65536 positions 0.5). Corrected within the loops, the scores
// cost every call of many rows 2 to 8%.
__device__ __forceinline__ float finiteOrNaN(float x) { return fmaf(x, 0.0f, x); }
__device__ __forceinline__ _Float16 finiteOrNaN(_Float16 x) { return __builtin_elementwise_fma(x, (_Float16)0.0f, x); }

// A kernel's parameters loaded again (it has no other arguments): a use of them that is hardly ever reached keeps no registers.
__device__ __forceinline__ FxParams paramsAgain() {
    auto p = (const __attribute__((address_space(4))) FxParams*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    FxParams a;
    __builtin_memcpy(&a, (const FxParams*)p, sizeof a);
    return a;
}

// The score of a row and a key; -infinity where the row does not see it.
template <int D, bool Q4>
__device__ __forceinline__ float plainScore(const FxParams& a, int kvh, const Row& row, int key) {
    const size_t meta = (size_t)kvh * a.key_row + key;
    const int pos = a.kpos ? a.kpos[meta] : key;
    const uint32_t mask = a.mask ? a.mask[(size_t)row.token * a.m_row2 + key] : 0u;
    if (pos < 0 || pos > row.limit || (a.kdoc && a.kdoc[meta] != row.doc) || mask == 0xFC00u) return -INFINITY;
    const float* q = a.q + (size_t)row.token * a.q_tok + (size_t)row.head * a.q_head;
    const char* k = a.k + (size_t)kvh * a.k_head + (size_t)key * a.k_row;
    float s = 0.0f;
    if constexpr (Q4) {
#pragma unroll 1
        for (int b = 0; b < D / 32; ++b, k += 18, q += 32) {
            const float d = halfBits(loadHalf(k));
#pragma unroll 4
            for (int e = 0; e < 16; ++e) {
                const int c = (unsigned char)k[2 + e];
                s = fmaf(q[e] * a.scale, d * (float)((c & 15) - 8), s);
                s = fmaf(q[e + 16] * a.scale, d * (float)((c >> 4) - 8), s);
            }
        }
    } else {
#pragma unroll 4
        for (int d = 0; d < D; ++d) s = fmaf(q[d] * a.scale, halfBits(loadHalf(k + 2 * d)), s);
    }
    if (a.softcap > 0.0f) s = a.softcap * tanhf(s / a.softcap);
    if (a.slopes) s = fmaf(-row.slope, fabsf((float)(row.pos - pos)), s);
    return a.mask ? s + halfBits(mask) : s;
}

// Row r over the tiles of TK keys sp, sp + splits, ..: values lane + 64 e of the sum of 2^(x - m) v to o, x the scores in base 2.
template <int D, bool Q4, int TK>
__device__ __forceinline__ void plainRow(const FxParams& a, int kvh, int r, int sp, int lane, float& m, float& l, float (&o)[D / 64]) {
    const Row row = rowOf(a, kvh, r);
    const char* vb = a.v + (size_t)kvh * a.v_head;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] = 0.0f;
    for (long long k0 = (long long)sp * TK; k0 < a.T; k0 += (long long)a.splits * TK) {
        const int key = (int)min(k0 + lane, (long long)a.T - 1);
        const float x = lane < TK && k0 + lane < a.T ? plainScore<D, Q4>(a, kvh, row, key) * kLog2e : -INFINITY;
        if (__any(!(x < INFINITY))) {  // infinity over infinity
            l = NAN;
            return;
        }
        const float top = fmaxf(m, waveMaxF(x));
        if (top == -INFINITY) continue;
        const float f = ex2(m - top), p = ex2(x - top);
        m = top;
        l = fmaf(l, f, waveSumF(p));
#pragma unroll
        for (int e = 0; e < D / 64; ++e) o[e] *= f;
        for (unsigned long long left = __ballot(p != 0.0f); left; left &= left - 1) {
            const int at = __builtin_ctzll(left);
            const float pk = __shfl(p, at);
            const char* v = vb + (size_t)(k0 + at) * a.v_row;
#pragma unroll
            for (int e = 0; e < D / 64; ++e) {
                const int d = lane + 64 * e;
                float y;
                if constexpr (Q4) {
                    const char* b = v + 18 * (d >> 5);
                    const int c = (unsigned char)b[2 + (d & 15)];
                    y = halfBits(loadHalf(b)) * (float)(((d & 16) ? c >> 4 : c & 15) - 8);
                } else {
                    y = halfBits(loadHalf(v + 2 * d));
                }
                o[e] = fmaf(pk, y, o[e]);
            }
        }
    }
}

}  // namespace fx

}  // namespace kcamd
