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
// integers; the scale d is applied to the f32 sums of each 32 keys' values (K), or split into d_hi (the seven
// leading bits of its significand) and d_lo (the other four), whose products with a code are exact in fp16
// (V): a third matrix chain instead of a rounded value.
#pragma once

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
typedef u4 u4a4 __attribute__((aligned(4)));
typedef u4 u4a2 __attribute__((aligned(2)));
typedef f32x4 f4a4 __attribute__((aligned(4)));
typedef __attribute__((address_space(3))) s4* LdsS4;
typedef __attribute__((address_space(3))) i2* LdsI2;

constexpr float kLog2e = 1.44269504088896f;
constexpr float kLn2 = 0.693147180559945f;
constexpr int kNoKey = INT_MAX;  // the position of a row past the cache's end or in an empty slot

// eight codes - 8 of a word as fp16, in the order of nibbles 0, 4, 1, 5, 2, 6, 3, 7: a nibble under the exponent of
// 1024 reads 1024 + code, so 1032 is subtracted (exact)
__device__ __forceinline__ h8 nibbles(uint32_t w) {
    h8 r;
    const h2 off = {(_Float16)1032.0f, (_Float16)1032.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const h2 x = __builtin_bit_cast(h2, ((w >> (4 * i)) & 0x000F000Fu) | 0x64006400u) - off;
        r[2 * i] = x[0];
        r[2 * i + 1] = x[1];
    }
    return r;
}
// the codes - 8 of a word's low (or, of w >> 4, high) nibbles as fp16, in the order of its bytes
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

// q values of one row as fp16 hi / lo parts: x 2^shift
struct QScale {
    int shift;
    float c;  // the factor that makes a sum of scaled products a score
};
__device__ __forceinline__ QScale qScale(float top, float scale) {
    const int e = top > 0.0f && top < INFINITY ? 8 - __builtin_amdgcn_frexp_expf(top) : 0;
    return {e, ldexpf(fabsf(scale), -e)};
}
__device__ __forceinline__ void qSplit(float x, bool neg, int shift, _Float16& hi, _Float16& lo) {
    const float y = ldexpf(neg ? -x : x, shift);
    hi = (_Float16)y;
    lo = (_Float16)(y - (float)hi);
}

// What a query row brings to its scores.
struct Row {
    int token, head;
    bool live;
    int limit;  // the last position it sees (causal), prefix included
    int pos, doc;
    float slope;
};
__device__ __forceinline__ Row rowOf(const FxParams& a, int kvh, int r) {
    Row w;
    w.live = r < a.rows;
    const int rr = w.live ? r : a.rows - 1;
    w.token = rr / a.G;
    w.head = kvh * a.G + (rr - w.token * a.G);
    w.pos = a.qpos ? a.qpos[w.token] : a.pos0 + w.token;
    w.limit = a.causal ? min(max(w.pos, a.prefix - 1), INT_MAX - 1) : INT_MAX - 1;
    w.doc = a.qdoc ? a.qdoc[w.token] : 0;
    w.slope = a.slopes ? a.slopes[w.head] : 0.0f;
    return w;
}

// tanh(x) = x P(x^2) / Q(x^2), the relative minimax fit of these degrees on |x| <= 9 (2e-8; beyond, tanh is 1 within
// 3e-8): a relative error of about 3e-7 over the whole range, where 1 - 2 / (exp(2x) + 1) would lose the small arguments
__device__ __forceinline__ float tanhFit(float x) {
    const float x0 = x;
    x = __builtin_amdgcn_fmed3f(x, -9.0f, 9.0f);
    const float u = x * x;
    float p = fmaf(u, 1.335463029050743e-08f, 2.0609057173714973e-05f);
    p = fmaf(u, p, 0.003495586570352316f);
    p = fmaf(u, p, 0.13381023705005646f);
    p = fmaf(u, p, 1.0f);
    float q = fmaf(u, 7.776545203341811e-07f, 0.00032856324105523527f);
    q = fmaf(u, q, 0.025876976549625397f);
    q = fmaf(u, q, 0.46714338660240173f);
    q = fmaf(u, q, 1.0f);
    return x0 == x0 ? x * p * __builtin_amdgcn_rcpf(q) : x0;
}

// A shaped score from the sum of scaled products: cap and distance (the mask's value and what is not seen come after).
struct Shape {
    float cap, inv_cap;
    bool bias;
};
__device__ __forceinline__ Shape shapeOf(const FxParams& a) {
    return {a.softcap, a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f, a.slopes != nullptr};
}

// exp2 on the transcendental unit: 0 below 2^-126, where the sums it joins do not see it
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }


__device__ __forceinline__ int waveMin(int x) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) x = min(x, __shfl_xor(x, o));
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int waveMax(int x) {
#pragma unroll
    for (int o = 1; o < 64; o *= 2) x = max(x, __shfl_xor(x, o));
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ float halfBits(uint32_t b) { return (float)__builtin_bit_cast(_Float16, (unsigned short)b); }
__device__ __forceinline__ uint32_t loadHalf(const char* p) { return *reinterpret_cast<const unsigned short*>(p); }


// ---- tiles of 32 keys x 32 rows (v_mfma_f32_32x32x16_f16; lane (j, h) = row j, lane half h)

// LDS bytes of a key's row as fp16: one pad chunk puts consecutive rows on different banks
template <int D>
constexpr int kKeyRow = 2 * D + 16;

// q as the B operand: values 16 ks + 8 h .. + 8 of the lane's row; returns the factor of its scores
template <int D>
__device__ __forceinline__ float loadRow32(const FxParams& a, const Row& row, int h, h8 (&qh)[D / 16], h8 (&ql)[D / 16]) {
    constexpr int KS = D / 16;
    const float* qp = a.q + (size_t)row.token * a.q_tok + (size_t)row.head * a.q_head + 8 * h;
    float x[KS][8], top = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const f32x4 u = *reinterpret_cast<const f4a4*>(qp + 16 * ks), w = *reinterpret_cast<const f4a4*>(qp + 16 * ks + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[ks][e] = u[e];
            x[ks][4 + e] = w[e];
            top = fmaxf(top, fmaxf(fabsf(u[e]), fabsf(w[e])));
        }
    }
    top = fmaxf(top, __shfl_xor(top, 32));
    const QScale qs = qScale(top, a.scale);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 hi, lo;
            qSplit(x[ks][e], a.scale < 0.0f, qs.shift, hi, lo);
            qh[ks][e] = hi;
            ql[ks][e] = lo;
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

// Sums of scaled products of the lane's 16 keys, 8 (v / 4) + 4 h + v % 4, from key rows in LDS (fp16 values, or codes - 8
// and f32 scales [block][key]).
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
            const float* ks = reinterpret_cast<const float*>(scales) + 32 * b + 4 * h;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 d = *reinterpret_cast<const f32x4*>(ks + 8 * g);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * g + e] = fmaf(d[e], s[4 * g + e], x[4 * g + e]);
            }
        }
    } else {
        f32x16 sh = zero, sl = zero;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const h8 ka = *reinterpret_cast<const h8*>(kr + 32 * ks);
            sh = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qh[ks], sh, 0, 0, 0);
            sl = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, ql[ks], sl, 0, 0, 0);
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = sh[v] + sl[v];
    }
}

// The mask's values of the lane's 16 keys of tile t.
struct MaskWords {
    uint32_t w[8];
    __device__ __forceinline__ void load(const unsigned short* mrow, int t, int h, int T) {
        const int words = (T + 1) / 2;
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
__device__ __forceinline__ float addMask(float x, uint32_t bits) { return bits == 0xFC00u ? -INFINITY : x + halfBits(bits); }

// Sums of products (times c) into shaped scores in base 2. meta (may be null): the tile's 32 positions and 32 document numbers
// in LDS; with it, what the row does not see becomes -infinity.
__device__ __forceinline__ void shapeScores(float (&x)[16], float c, const Shape& shape, const Row& row, const int* meta,
                                            const MaskWords* mk, int t, int h) {
#pragma unroll
    for (int v = 0; v < 16; ++v) x[v] *= c;
    if (shape.cap > 0.0f) {
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = shape.cap * tanhFit(x[v] * shape.inv_cap);
    }
    if (shape.bias) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            int4 kp = {};
            if (meta) kp = *reinterpret_cast<const int4*>(meta + 8 * g + 4 * h);
            const int p[4] = {kp.x, kp.y, kp.z, kp.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                x[4 * g + e] = fmaf(-row.slope, fabsf((float)(row.pos - (meta ? p[e] : t * 32 + 8 * g + 4 * h + e))), x[4 * g + e]);
        }
    }
    if (mk) {
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = addMask(x[v], (v & 1) ? mk->w[v >> 1] >> 16 : mk->w[v >> 1] & 0xFFFFu);
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) x[v] *= kLog2e;
    if (meta) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int4 kp = *reinterpret_cast<const int4*>(meta + 8 * g + 4 * h);
            const int4 kd = *reinterpret_cast<const int4*>(meta + 32 + 8 * g + 4 * h);
            const int p[4] = {kp.x, kp.y, kp.z, kp.w}, dd[4] = {kd.x, kd.y, kd.z, kd.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * g + e] = p[e] <= row.limit && dd[e] == row.doc ? x[4 * g + e] : -INFINITY;
        }
    }
}

}  // namespace fx

}  // namespace kcamd
