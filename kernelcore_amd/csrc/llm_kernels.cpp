// llm_kernels.cpp -- the built-in kernel table: argument validation and launch per kernel name.
//
// Validation keeps the reference's rules (arasheedu/Kernelcore llm/llm_kernels.cpp): sizes must
// be positive and fit int32 indexing, every buffer must lie inside one live allocation, and the
// shape rules of each kernel (rows % 8, k % 256, ...) hold. A rejected launch returns
// InvalidValue or InvalidPointer with a detail text, as there. The System V marshalling, chunk
// planning and CPU executor are replaced by one HIP grid per launch (launch.hpp).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <numeric>

#include "internal.hpp"
#include "kflash_ext.hpp"
#include "kquant.hpp"
#include "launch.hpp"
#include "kquantize.hpp"
#include "kdecode.hpp"
#include "kserve.hpp"
#include "kv_cache.hpp"
#include "model_kernels.hpp"

namespace {

using kcamd::checkRange;
using kcamd::setDetail;

constexpr int64_t kMaxIndex = INT32_MAX;

bool fitsIndex(int64_t a, int64_t b = 1) { return a >= 0 && b >= 0 && (b == 0 || a <= kMaxIndex / b); }
size_t f32Bytes(int64_t n) { return static_cast<size_t>(n) * sizeof(float); }
size_t i32Bytes(int64_t n) { return static_cast<size_t>(n) * sizeof(int); }

#define KC_TRY(expr)                 \
    do {                             \
        if (int e_ = (expr)) return e_; \
    } while (0)

int invalid(const char* what) {
    setDetail("%s", what);
    return KC_ERROR_INVALID_VALUE;
}

// Optional device dims array: a live allocation of n ints whose known host copy matches `want`.
int checkDims(const int* dims, const int* want, int n) {
    if (!dims) return 0;
    KC_TRY(checkRange(dims, i32Bytes(n), "dims"));
    if (!kcamd::dimsAgree(dims, want, n)) return KC_ERROR_INVALID_VALUE;
    return 0;
}

hipStream_t hs(void* s) { return static_cast<hipStream_t>(s); }

// ---- vector_add (adapters/vector_add_adapter.cpp:14-24)

int vectorAddValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcVectorAddArgs*>(p);
    if (a.count < 0) return invalid("count < 0");
    const size_t bytes = f32Bytes(a.count);
    KC_TRY(checkRange(a.a, bytes, "a"));
    KC_TRY(checkRange(a.b, bytes, "b"));
    KC_TRY(checkRange(a.out, bytes, "out"));
    return 0;
}
int vectorAddLaunch(const void* p, void* s) {
    const auto& a = *static_cast<const kcVectorAddArgs*>(p);
    return kcamd::launchVectorAdd(a.a, a.b, a.out, a.count, hs(s));
}

// ---- quantize_q8x4 (llm_kernels.cpp:180-189)

int quantValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcQuantizeArgs*>(p);
    if (a.count < 0 || !fitsIndex(a.count, 32)) return invalid("count out of range");
    KC_TRY(checkRange(a.x, f32Bytes(int64_t(a.count) * 32), "x"));
    KC_TRY(checkRange(a.xq, i32Bytes(int64_t(a.count) * 8), "xq"));
    KC_TRY(checkRange(a.xd, f32Bytes(int64_t(a.count) * 2), "xd"));
    return 0;
}
int quantLaunch(const void* p, void* s) {
    const auto& a = *static_cast<const kcQuantizeArgs*>(p);
    return kcamd::launchQuantizeQ8x4(a.x, a.xq, a.xd, a.count, hs(s));
}

// ---- matvec_q4k_q8 / matvec_q6k_q8 (llm_kernels.cpp:264-279: kquantMarshal)

template <bool Q6>
int kquantValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcMatvecQ4Q8Args*>(p);
    if (a.rows < 0 || a.rows % 8 != 0 || a.k <= 0 || a.k % 256 != 0 || !fitsIndex(a.rows, a.k))
        return invalid("rows must be a non-negative multiple of 8 and k a positive multiple of 256");
    if (a.k > kcamd::kMatvecMaxK) return invalid("k exceeds the matvec's activation staging (32768)");
    const int64_t nb = a.k / 32;
    if (reinterpret_cast<uintptr_t>(a.qw) % 16) return invalid("qw (a weight stream) must be 16-byte aligned");
    KC_TRY(checkRange(a.qw, kcamd::streamBytes(Q6, a.rows, a.k), "qw"));
    KC_TRY(checkRange(a.xq, i32Bytes(nb * 8), "xq"));
    KC_TRY(checkRange(a.xd, f32Bytes(nb * 2), "xd"));
    KC_TRY(checkRange(a.y, f32Bytes(a.rows), "y"));
    const int want[2] = {a.rows, a.k};
    return checkDims(a.dims, want, 2);
}
template <bool Q6>
int kquantLaunch(const void* p, void* s) {
    return kcamd::launchMatvecKq(Q6, *static_cast<const kcMatvecQ4Q8Args*>(p), hs(s));
}

// ---- matmul_{q4k,q6k}_q8{,k}x{4,8} (llm_kernels.cpp:290-312: matmulKMarshal)

template <bool Q6, bool K8>
int matmulValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcMatmulKQ8Args*>(p);
    if (a.rows <= 0 || a.rows % 8 != 0 || a.k <= 0 || a.k % 256 != 0 || a.ncols <= 0 || a.row_block <= 0 ||
        !fitsIndex(a.rows, a.k))
        return invalid("rows must be a positive multiple of 8, k a positive multiple of 256, ncols and row_block > 0");
    const int64_t slot = K8 ? int64_t(a.k / 256) * 85 : int64_t(a.k / 32) * 11;
    if (!fitsIndex(slot, a.ncols) || !fitsIndex(a.rows, a.ncols) || a.ncols > 65535 * 8)
        return invalid("ncols out of range");
    if (reinterpret_cast<uintptr_t>(a.qw) % 16) return invalid("qw (a weight stream) must be 16-byte aligned");
    KC_TRY(checkRange(a.qw, kcamd::streamBytes(Q6, a.rows, a.k), "qw"));
    KC_TRY(checkRange(a.xq, i32Bytes(slot * a.ncols), "xq"));
    KC_TRY(checkRange(a.y, f32Bytes(int64_t(a.rows) * a.ncols), "y"));
    const int want[4] = {a.rows, a.k, a.ncols, a.row_block};
    return checkDims(a.dims, want, 4);
}
template <bool Q6, bool K8>
int matmulLaunch(const void* p, void* s) {
    return kcamd::launchMatmulKq(Q6, K8, *static_cast<const kcMatmulKQ8Args*>(p), hs(s));
}

// ---- matmul_f16 (llm_kernels.cpp:834-847: matmulF16Marshal). The reference's thread-count
// limit (rows x column tiles of 4 below 2^24, a CPU chunking bound) is kept so that the same
// launches are accepted.

int matmulF16Validate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcMatmulF16Args*>(p);
    if (a.rows <= 0 || a.rows % 8 || a.k <= 0 || a.k % 2 || a.ncols <= 0 || !fitsIndex(a.rows, a.k) ||
        !fitsIndex(a.ncols, std::max(a.rows, a.k)) || int64_t(a.rows) * ((a.ncols + 3) / 4) >= (int64_t(1) << 24))
        return invalid("rows must be a positive multiple of 8, k positive and even, ncols positive");
    if (reinterpret_cast<uintptr_t>(a.qw) % 4 || reinterpret_cast<uintptr_t>(a.x) % 4 ||
        reinterpret_cast<uintptr_t>(a.y) % 4)
        return invalid("qw, x and y must be 4-byte aligned");
    KC_TRY(checkRange(a.qw, i32Bytes(int64_t(a.rows) * (a.k / 2)), "qw"));
    KC_TRY(checkRange(a.x, f32Bytes(int64_t(a.ncols) * a.k), "x"));
    KC_TRY(checkRange(a.y, f32Bytes(int64_t(a.ncols) * a.rows), "y"));
    const int want[3] = {a.rows, a.k, a.ncols};
    return checkDims(a.dims, want, 3);
}
int matmulF16Launch(const void* p, void* s) {
    const auto& a = *static_cast<const kcMatmulF16Args*>(p);
    return kcamd::launchMatmulF16(a.qw, a.x, a.y, a.rows, a.k, a.ncols, hs(s));
}

// ---- quantize_cols / quantize_cols_k (llm_kernels.cpp:331-345: quantColsMarshal)

template <int kBlock>
int quantColsValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcQuantizeColsArgs*>(p);
    const int64_t slot = kBlock == 32 ? int64_t(a.k / 32) * 11 : int64_t(a.k / 256) * 85;
    if (a.k <= 0 || a.k % 256 != 0 || a.ncols <= 0 || !fitsIndex(a.k, a.ncols) || !fitsIndex(slot, a.ncols))
        return invalid("k must be a positive multiple of 256 and ncols positive");
    KC_TRY(checkRange(a.x, f32Bytes(int64_t(a.k) * a.ncols), "x"));
    KC_TRY(checkRange(a.q, i32Bytes(slot * a.ncols), "q"));
    const int want[2] = {a.k / kBlock, a.ncols};
    return checkDims(a.dims, want, 2);
}
template <int kBlock>
int quantColsLaunch(const void* p, void* s) {
    const auto& a = *static_cast<const kcQuantizeColsArgs*>(p);
    if (kBlock == 32) return kcamd::launchQuantizeCols(a.x, a.q, a.k, a.ncols, hs(s));
    return kcamd::launchQuantizeColsK(a.x, a.q, a.k, a.ncols, hs(s));
}

// ---- ggml layer fusions (llm_kernels.cpp:402-570: checkRowsQ, normDimsOk and the marshals)

int checkRowsQ(int n, int rows, const int* q) {
    if (n <= 0 || n % 256 || rows <= 0 || !fitsIndex(n, rows) || int64_t(n) * rows >= (1 << 24))
        return invalid("n must be a positive multiple of 256, rows positive, n * rows < 2^24");
    return checkRange(q, i32Bytes(int64_t(rows) * (n / 32) * 11), "q");
}

int addSumsqValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcAddSumsqFArgs*>(p);
    KC_TRY(checkRowsQ(a.n, a.rows, a.q));
    const size_t bytes = f32Bytes(int64_t(a.n) * a.rows);
    KC_TRY(checkRange(a.a, bytes, "a"));
    KC_TRY(checkRange(a.b, bytes, "b"));
    KC_TRY(checkRange(a.out, bytes, "out"));
    const int want[3] = {a.n / 32, a.n, a.rows};
    return checkDims(a.dims, want, 3);
}
int addSumsqLaunch(const void* p, void* s) {
    const auto& a = *static_cast<const kcAddSumsqFArgs*>(p);
    return kcamd::launchAddSumsq(a.a, a.b, a.out, a.q, a.n, a.rows, hs(s));
}

int sumsqValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcSumsqPartArgs*>(p);
    KC_TRY(checkRowsQ(a.n, a.rows, a.q));
    KC_TRY(checkRange(a.x, f32Bytes(int64_t(a.n) * a.rows), "x"));
    const int want[3] = {a.n / 32, a.n, a.rows};
    return checkDims(a.dims, want, 3);
}
int sumsqLaunch(const void* p, void* s) {
    const auto& a = *static_cast<const kcSumsqPartArgs*>(p);
    return kcamd::launchAddSumsq(nullptr, a.x, nullptr, a.q, a.n, a.rows, hs(s));
}

template <bool K8>
int normMulValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcNormMulQ8Args*>(p);
    if (K8) {
        if (a.n <= 0 || a.n % 256 || a.rows <= 0 || int64_t(a.n) * a.rows >= (1 << 24))
            return invalid("n must be a positive multiple of 256, rows positive, n * rows < 2^24");
        KC_TRY(checkRange(a.q, i32Bytes(int64_t(a.rows) * (a.n / 256 * 85 + a.n / 32 * 11)), "q"));
    } else {
        KC_TRY(checkRowsQ(a.n, a.rows, a.q));
    }
    const size_t bytes = f32Bytes(int64_t(a.n) * a.rows);
    KC_TRY(checkRange(a.x, bytes, "x"));
    KC_TRY(checkRange(a.w, f32Bytes(a.n), "w"));
    KC_TRY(checkRange(a.y, bytes, "y"));
    if (K8) {
        const int want[4] = {a.n / 256, a.n, a.rows, a.rows * (a.n / 256 * 85)};
        return checkDims(a.dims, want, 4);
    }
    const int want[3] = {a.n / 32, a.n, a.rows};
    return checkDims(a.dims, want, 3);
}
template <bool K8>
int normMulLaunch(const void* p, void* s) {
    return kcamd::launchNormMulQ8(K8, *static_cast<const kcNormMulQ8Args*>(p), hs(s));
}

int addNormValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcAddNormQ8FArgs*>(p);
    KC_TRY(checkRowsQ(a.n, a.rows, a.q));
    if (a.n > 8192) return invalid("add_norm_q8_f: rows of at most 8192 values");
    if ((a.a != nullptr) != (a.b != nullptr)) return invalid("a and b are both given or both null");
    const size_t bytes = f32Bytes(int64_t(a.n) * a.rows);
    if (a.a) {
        KC_TRY(checkRange(a.a, bytes, "a"));
        KC_TRY(checkRange(a.b, bytes, "b"));
    }
    KC_TRY(checkRange(a.x, bytes, "x"));
    KC_TRY(checkRange(a.w, f32Bytes(a.n), "w"));
    KC_TRY(checkRange(a.y, bytes, "y"));
    const int want[3] = {a.n / 32, a.n, a.rows};
    return checkDims(a.dims, want, 3);
}
int addNormLaunch(const void* p, void* s) {
    const auto& a = *static_cast<const kcAddNormQ8FArgs*>(p);
    return kcamd::launchAddNormQ8(a.a, a.b, a.x, a.w, a.y, a.q, a.n, a.rows, a.eps, hs(s));
}

template <bool K8>
int siluQValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcSiluMulQ8FArgs*>(p);
    if (a.n <= 0 || a.n % 256 || a.cols <= 0 || int64_t(a.n) * a.cols >= (1 << 24))
        return invalid("n must be a positive multiple of 256, cols positive, n * cols < 2^24");
    KC_TRY(checkRange(a.q, i32Bytes(int64_t(a.cols) * (K8 ? a.n / 256 * 85 : a.n / 32 * 11)), "q"));
    const size_t bytes = f32Bytes(int64_t(a.n) * a.cols);
    KC_TRY(checkRange(a.g, bytes, "g"));
    KC_TRY(checkRange(a.u, bytes, "u"));
    KC_TRY(checkRange(a.y, bytes, "y"));
    const int want[2] = {a.n, a.cols};
    return checkDims(a.dims, want, 2);
}
template <bool K8>
int siluQLaunch(const void* p, void* s) {
    return kcamd::launchSiluMulQ8(K8, *static_cast<const kcSiluMulQ8FArgs*>(p), hs(s));
}

// ---- rms_norm, mul_rows, silu_mul, rope_ggml, set_rows_f16 (llm_kernels.cpp:386-400, 616-631, 944-972)

int rmsValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcRmsNormArgs*>(p);
    if (a.n <= 0 || a.rows < 0 || !fitsIndex(a.rows, a.n)) return invalid("n must be positive, rows >= 0");
    const size_t bytes = f32Bytes(int64_t(a.rows) * a.n);
    KC_TRY(checkRange(a.x, bytes, "x"));
    KC_TRY(checkRange(a.w, f32Bytes(a.n), "w"));
    return checkRange(a.y, bytes, "y");
}
int rmsLaunch(const void* p, void* s) { return kcamd::launchRmsNorm(*static_cast<const kcRmsNormArgs*>(p), hs(s)); }

int mulRowsValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcMulRowsArgs*>(p);
    if (a.n <= 0 || a.n % 8 || a.count < 0 || a.count % a.n) return invalid("n must be a positive multiple of 8 dividing count");
    KC_TRY(checkRange(a.x, f32Bytes(a.count), "x"));
    KC_TRY(checkRange(a.w, f32Bytes(a.n), "w"));
    return checkRange(a.y, f32Bytes(a.count), "y");
}
int mulRowsLaunch(const void* p, void* s) { return kcamd::launchMulRows(*static_cast<const kcMulRowsArgs*>(p), hs(s)); }

int siluValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcSiluMulArgs*>(p);
    if (a.count < 0) return invalid("count < 0");
    const size_t bytes = f32Bytes(a.count);
    KC_TRY(checkRange(a.g, bytes, "g"));
    KC_TRY(checkRange(a.u, bytes, "u"));
    return checkRange(a.out, bytes, "out");
}
int siluLaunch(const void* p, void* s) { return kcamd::launchSiluMul(*static_cast<const kcSiluMulArgs*>(p), hs(s)); }

int ropeValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcRopeGgmlArgs*>(p);
    if (a.head_dim <= 0 || a.head_dim % 16 || a.n_head <= 0 || a.n_tokens < 0)
        return invalid("head_dim must be a positive multiple of 16, n_head positive, n_tokens >= 0");
    const int64_t pairs = a.head_dim / 2, count = pairs * a.n_head * a.n_tokens;
    if (!fitsIndex(count, 2)) return invalid("too many values");
    KC_TRY(checkRange(a.x, f32Bytes(count * 2), "x"));
    KC_TRY(checkRange(a.y, f32Bytes(count * 2), "y"));
    KC_TRY(checkRange(a.pos, i32Bytes(a.n_tokens), "pos"));
    KC_TRY(checkRange(a.ff, f32Bytes(pairs), "ff"));
    const int want[5] = {(int)pairs, a.n_head, (int)(pairs * a.n_tokens), a.neox ? 1 : 2, a.neox ? (int)pairs : 1};
    return checkDims(a.dims, want, 5);
}
int ropeLaunch(const void* p, void* s) { return kcamd::launchRope(*static_cast<const kcRopeGgmlArgs*>(p), hs(s)); }

int setRowsValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcSetRowsF16Args*>(p);
    if (a.pairs <= 0 || a.pairs % 8 || a.rows <= 0 || a.dst_rows <= 0 || a.src_row < 2 * a.pairs ||
        a.dst_row < a.pairs || int64_t(a.pairs) * a.rows >= (1 << 24) || !fitsIndex(a.rows, a.src_row) ||
        !fitsIndex(a.dst_rows, a.dst_row))
        return invalid("set_rows_f16 shape");
    KC_TRY(checkRange(a.src, f32Bytes(int64_t(a.rows - 1) * a.src_row + 2 * a.pairs), "src"));
    KC_TRY(checkRange(a.idx, i32Bytes(int64_t(a.rows) * 2), "idx"));
    KC_TRY(checkRange(a.dst, i32Bytes(int64_t(a.dst_rows) * a.dst_row), "dst"));
    const int want[5] = {a.pairs, a.rows, a.src_row, a.dst_row, a.dst_rows};
    return checkDims(a.dims, want, 5);
}
int setRowsLaunch(const void* p, void* s) { return kcamd::launchSetRows(*static_cast<const kcSetRowsF16Args*>(p), hs(s)); }

// ---- FLASH_ATTN_EXT: fa_scores, fa_max, fa_exp, fa_values (llm_kernels.cpp:972-1013) and the fused form

int faShape(const kcFaDims& d, const int* dims) {
    if (d.H <= 0 || d.T <= 0 || d.D <= 0 || d.D % 8 || d.H_kv <= 0 || d.group <= 0 || d.H != d.H_kv * d.group ||
        d.N <= 0 || d.tp % 8 || d.tp < d.T || d.k_row < 0 || d.k_head < 0 || d.v_row < 0 || d.v_head < 0 ||
        d.q_tok < 0 || d.q_head < d.D || d.m_row < 0 || (d.has_mask != 0 && d.has_mask != 1))
        return invalid("FaDims out of range");
    const int64_t cap = 1 << 24;
    if (!fitsIndex(int64_t(d.H) * d.N, d.tp) || int64_t(d.H) * d.N * d.tp >= cap || int64_t(d.N) * d.H * d.D >= cap ||
        !fitsIndex(d.T, std::max(d.k_row, d.v_row)) || !fitsIndex(d.N, std::max(d.q_tok, d.m_row)) ||
        !fitsIndex(d.H, d.q_head))
        return invalid("FaDims too large");
    const int want[15] = {d.H, d.T, d.D, d.group, d.tp, d.k_row, d.k_head, d.v_row, d.v_head, d.N, d.q_tok, d.q_head,
                          d.m_row, d.has_mask, d.H_kv};
    return checkDims(dims, want, 15);
}
size_t faScoreBytes(const kcFaDims& d) { return f32Bytes(int64_t(d.H) * d.N * d.tp); }
size_t faCacheBytes(const kcFaDims& d, int row, int head) {
    return (size_t(d.T - 1) * size_t(row) + size_t(d.H_kv - 1) * size_t(head) + size_t(d.D / 2)) * sizeof(int);
}
int faQMask(const kcFaDims& d, const float* q, const int* mask) {
    KC_TRY(checkRange(q, f32Bytes(int64_t(d.N - 1) * d.q_tok + int64_t(d.H - 1) * d.q_head + d.D), "q"));
    if (d.has_mask) return checkRange(mask, (size_t(d.N - 1) * size_t(d.m_row) + size_t(d.T + 1) / 2) * sizeof(int), "mask");
    return 0;
}

int faScoresValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcFaScoresArgs*>(p);
    KC_TRY(faShape(a.d, a.dims));
    KC_TRY(faQMask(a.d, a.q, a.mask));
    KC_TRY(checkRange(a.k, faCacheBytes(a.d, a.d.k_row, a.d.k_head), "k"));
    return checkRange(a.s, faScoreBytes(a.d), "s");
}
int faScoresLaunch(const void* p, void* s) { return kcamd::launchFaScores(*static_cast<const kcFaScoresArgs*>(p), hs(s)); }

int faMaxValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcFaMaxArgs*>(p);
    KC_TRY(faShape(a.d, a.dims));
    KC_TRY(checkRange(a.s, faScoreBytes(a.d), "s"));
    return checkRange(a.m, f32Bytes(int64_t(a.d.H) * a.d.N), "m");
}
int faMaxLaunch(const void* p, void* s) { return kcamd::launchFaMax(*static_cast<const kcFaMaxArgs*>(p), hs(s)); }

int faExpValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcFaExpArgs*>(p);
    KC_TRY(faShape(a.d, a.dims));
    KC_TRY(checkRange(a.s, faScoreBytes(a.d), "s"));
    return checkRange(a.m, f32Bytes(int64_t(a.d.H) * a.d.N), "m");
}
int faExpLaunch(const void* p, void* s) { return kcamd::launchFaExp(*static_cast<const kcFaExpArgs*>(p), hs(s)); }

int faValuesValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcFaValuesArgs*>(p);
    KC_TRY(faShape(a.d, a.dims));
    KC_TRY(checkRange(a.p, faScoreBytes(a.d), "p"));
    KC_TRY(checkRange(a.v, faCacheBytes(a.d, a.d.v_row, a.d.v_head), "v"));
    return checkRange(a.out, f32Bytes(int64_t(a.d.N) * a.d.H * a.d.D), "out");
}
int faValuesLaunch(const void* p, void* s) { return kcamd::launchFaValues(*static_cast<const kcFaValuesArgs*>(p), hs(s)); }

int flashValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcFlashAttnArgs*>(p);
    KC_TRY(faShape(a.d, a.dims));
    if (a.d.T > kcamd::kFlashAttnMaxT) return invalid("flash_attn_f16: T exceeds 16384 (use the fa_* kernels)");
    KC_TRY(faQMask(a.d, a.q, a.mask));
    KC_TRY(checkRange(a.k, faCacheBytes(a.d, a.d.k_row, a.d.k_head), "k"));
    KC_TRY(checkRange(a.v, faCacheBytes(a.d, a.d.v_row, a.d.v_head), "v"));
    return checkRange(a.out, f32Bytes(int64_t(a.d.N) * a.d.H * a.d.D), "out");
}
int flashLaunch(const void* p, void* s) { return kcamd::launchFlashAttn(*static_cast<const kcFlashAttnArgs*>(p), hs(s)); }

int flashDecodeValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcFlashDecodeArgs*>(p);
    KC_TRY(faShape(a.d, a.dims));
    if (!kcamd::flashDecodeSupports(a.d.D, a.d.group)) return invalid("flash_decode_f16: D must be 64 or 128, group at most 8");
    if (a.d.q_head % 4 || a.d.q_tok % 4) return invalid("flash_decode_f16: q rows and heads at 16-byte strides");
    KC_TRY(faQMask(a.d, a.q, a.mask));
    KC_TRY(checkRange(a.k, faCacheBytes(a.d, a.d.k_row, a.d.k_head), "k"));
    KC_TRY(checkRange(a.v, faCacheBytes(a.d, a.d.v_row, a.d.v_head), "v"));
    KC_TRY(checkRange(a.part, kcamd::flashDecodePartFloats(a.d) * sizeof(float), "part"));
    return checkRange(a.out, f32Bytes(int64_t(a.d.N) * a.d.H * a.d.D), "out");
}
int flashDecodeLaunch(const void* p, void* s) {
    return kcamd::launchFlashDecode(*static_cast<const kcFlashDecodeArgs*>(p), hs(s));
}

// ---- repack_kquant / unpack_kquant: ggml blocks <-> this device's weight stream

template <bool Unpack>
int repackValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcKquantRepackArgs*>(p);
    if (a.qtype != KC_QTYPE_Q4_K && a.qtype != KC_QTYPE_Q6_K) return invalid("qtype must be Q4_K (12) or Q6_K (14)");
    if (a.rows < 0 || a.k <= 0 || a.k % 256 != 0 || !fitsIndex(a.rows, a.k))
        return invalid("rows must be non-negative and k a positive multiple of 256");
    const bool q6 = a.qtype == KC_QTYPE_Q6_K;
    const size_t ggml = size_t(a.rows) * size_t(a.k / 256) * (q6 ? kcamd::kQ6kBlock : kcamd::kQ4kBlock);
    const size_t stream = kcamd::streamBytes(q6, a.rows, a.k);
    KC_TRY(checkRange(a.src, Unpack ? stream : ggml, "src"));
    KC_TRY(checkRange(a.dst, Unpack ? ggml : stream, "dst"));
    return 0;
}
template <bool Unpack>
int repackLaunch(const void* p, void* s) {
    return kcamd::launchRepack(*static_cast<const kcKquantRepackArgs*>(p), Unpack, hs(s));
}

// ---- get_rows_kquant (llm/llm_reference.cpp:342-383, used by llm/gguf_model.cpp:96-104)

int getRowsValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcGetRowsKquantArgs*>(p);
    if (a.qtype != KC_QTYPE_Q4_K && a.qtype != KC_QTYPE_Q6_K) return invalid("qtype must be Q4_K (12) or Q6_K (14)");
    if (a.rows < 0 || a.n < 0 || a.k <= 0 || a.k % 256 != 0 || !fitsIndex(a.rows, a.k) || !fitsIndex(a.n, a.k))
        return invalid("rows and n must be non-negative and k a positive multiple of 256");
    KC_TRY(checkRange(a.qw, kcamd::streamBytes(a.qtype == KC_QTYPE_Q6_K, a.rows, a.k), "qw"));
    KC_TRY(checkRange(a.ids, i32Bytes(a.n), "ids"));
    return checkRange(a.y, f32Bytes(int64_t(a.n) * a.k), "y");
}
int getRowsLaunch(const void* p, void* s) {
    const auto& a = *static_cast<const kcGetRowsKquantArgs*>(p);
    return kcamd::launchGetRows(a.qtype == KC_QTYPE_Q6_K, a.qw, a.ids, a.y, a.n, a.k, a.rows, hs(s));
}

// ---- operators over a key/value cache: set_rows_q4_0, get_rows_q4_0, flash_ext_*, attn_weights_*, kv_keep, kv_gather

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
// Bytes from the first of n rows `row` bytes apart to the end of the last one's `bytes`; false past 2^62.
bool extent(int64_t n, int64_t row, int64_t bytes, int64_t* out) {
    if (n <= 0) {
        *out = 0;
        return true;
    }
    int64_t x;
    if (row < 0 || __builtin_mul_overflow(n - 1, row, &x) || __builtin_add_overflow(x, bytes, &x) || x > (int64_t(1) << 62)) return false;
    *out = x;
    return true;
}

int setRowsQ40Validate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcSetRowsQ40Args*>(p);
    int64_t src, dst;
    if (a.n <= 0 || a.n % 32 || a.rows < 0 || a.rows > 65535 * 8 || a.src_row < a.n || a.dst_rows < 0 || a.dst_row < a.n / 32 * 18 ||
        a.dst_row % 2 || !extent(a.rows, a.src_row, a.n, &src) || !extent(a.dst_rows, a.dst_row, a.n / 32 * 18, &dst))
        return invalid("set_rows_q4_0: n a positive multiple of 32, rows of at least n values, dst_row even");
    if (!aligned(a.src, 4) || !aligned(a.idx, 4) || !aligned(a.dst, 2)) return invalid("set_rows_q4_0: src and idx 4-byte, dst 2-byte aligned");
    KC_TRY(checkRange(a.src, size_t(src) * 4, "src"));
    KC_TRY(checkRange(a.idx, size_t(a.rows) * 8, "idx"));
    return checkRange(a.dst, size_t(dst), "dst");
}
int setRowsQ40Launch(const void* p, void* s) { return kcamd::launchSetRowsQ40(*static_cast<const kcSetRowsQ40Args*>(p), hs(s)); }

int getRowsQ40Validate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcGetRowsQ40Args*>(p);
    int64_t src;
    if (a.n <= 0 || a.n % 32 || a.rows < 0 || a.src_rows < 0 || a.src_row < a.n / 32 * 18 || a.src_row % 2 ||
        !extent(a.src_rows, a.src_row, a.n / 32 * 18, &src))
        return invalid("get_rows_q4_0: n a positive multiple of 32, rows of at least n values, src_row even");
    if (!aligned(a.src, 2) || !aligned(a.idx, 4) || !aligned(a.y, 4)) return invalid("get_rows_q4_0: idx and y 4-byte, src 2-byte aligned");
    KC_TRY(checkRange(a.src, size_t(src), "src"));
    KC_TRY(checkRange(a.idx, size_t(a.rows) * 8, "idx"));
    return checkRange(a.y, size_t(a.rows) * size_t(a.n) * 4, "y");
}
int getRowsQ40Launch(const void* p, void* s) { return kcamd::launchGetRowsQ40(*static_cast<const kcGetRowsQ40Args*>(p), hs(s)); }

// The sizes alone (no pointers): what kcFlashExtPartBytes accepts too.
int fxShape(const kcFlashExtDims& d) {
    if (d.H <= 0 || d.H_kv <= 0 || d.H % d.H_kv || d.H_kv > 65535 || (d.D != 64 && d.D != 128 && d.D != 256) || d.N < 0 || d.T < 0 ||
        d.T > INT32_MAX - 1024)  // (the kernels count positions in 32 bits, up to 512 past the last one)
        return invalid("flash_ext: H a positive multiple of H_kv, D 64, 128 or 256, N and T not negative, T below 2^31 - 1024");
    if (d.q_tok < 0 || d.q_head < 0 || d.m_row < 0 || d.key_row < 0 || d.k_row < 0 || d.k_head < 0 || d.v_row < 0 || d.v_head < 0)
        return invalid("flash_ext: negative strides");
    if ((d.causal != 0 && d.causal != 1) || d.prefix < 0) return invalid("flash_ext: causal 0 or 1, prefix not negative");
    if (d.pos0 < 0 || int64_t(d.pos0) + d.N >= INT32_MAX) return invalid("flash_ext: positions from 0 to 2^31 - 2");
    const int64_t rows = int64_t(d.N) * (d.H / d.H_kv);
    if (rows * d.H_kv * d.D > INT32_MAX || (rows + 127) / 128 > 65535) return invalid("flash_ext: too many query rows");
    return 0;
}
int fxCache(const kcFlashExtDims& d, bool q4, const void* p, int64_t row, int64_t head, const char* what) {
    const int64_t bytes = q4 ? d.D / 32 * 18 : d.D * 2, unit = q4 ? 2 : 4;
    int64_t a, b;
    if (row % unit || head % unit || !aligned(p, size_t(unit)))
        return invalid(q4 ? "flash_ext: Q4_0 rows, heads and base at multiples of 2 bytes" : "flash_ext: fp16 rows, heads and base at multiples of 4 bytes");
    if (!extent(d.H_kv, head, bytes, &a) || !extent(d.T, row, a, &b)) return invalid("flash_ext: strides too large");
    return checkRange(p, size_t(b), what);
}
int fxInputs(const kcFlashExtDims& d, bool q4, const float* q, const void* k, const int* mask, const int* qpos, const int* kpos,
             const int* qdoc, const int* kdoc, const float* slopes, float scale, float softcap) {
    KC_TRY(fxShape(d));
    // (caps whose reciprocals and products with scores keep their bits in f32)
    if (!(scale == scale) || scale - scale != 0.0f || !(softcap == 0.0f || (softcap >= 0x1p-100f && softcap <= 0x1p100f)))
        return invalid("flash_ext: scale finite, softcap 0 or from 2^-100 to 2^100");
    if ((qdoc != nullptr) != (kdoc != nullptr)) return invalid("flash_ext: qdoc and kdoc are both given or both null");
    if (d.key_row && d.key_row < d.T && d.H_kv > 1) return invalid("flash_ext: key_row is 0 or at least T");
    if (!aligned(q, 4) || !aligned(mask, 4) || !aligned(qpos, 4) || !aligned(kpos, 4) || !aligned(qdoc, 4) || !aligned(kdoc, 4) ||
        !aligned(slopes, 4))
        return invalid("flash_ext: 4-byte aligned arrays");
    int64_t x, y;
    if (!extent(d.H, d.q_head, d.D, &x) || !extent(d.N, d.q_tok, x, &y)) return invalid("flash_ext: q strides too large");
    KC_TRY(checkRange(q, size_t(y) * 4, "q"));
    KC_TRY(fxCache(d, q4, k, d.k_row, d.k_head, "k"));
    if (mask && d.N && d.T) {
        if (d.m_row < (int64_t(d.T) + 1) / 2) return invalid("flash_ext: mask rows hold T values");
        KC_TRY(checkRange(mask, (size_t(d.N - 1) * size_t(d.m_row) + (size_t(d.T) + 1) / 2) * 4, "mask"));
    }
    const size_t keys = d.T ? (size_t(d.H_kv - 1) * size_t(d.key_row) + size_t(d.T)) * 4 : 0;
    if (qpos) KC_TRY(checkRange(qpos, size_t(d.N) * 4, "qpos"));
    if (qdoc) KC_TRY(checkRange(qdoc, size_t(d.N) * 4, "qdoc"));
    if (kpos) KC_TRY(checkRange(kpos, keys, "kpos"));
    if (kdoc) KC_TRY(checkRange(kdoc, keys, "kdoc"));
    if (slopes) KC_TRY(checkRange(slopes, size_t(d.H) * 4, "slopes"));
    return 0;
}

template <bool Q4>
int flashExtValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcFlashExtArgs*>(p);
    KC_TRY(fxInputs(a.d, Q4, a.q, a.k, a.mask, a.qpos, a.kpos, a.qdoc, a.kdoc, a.slopes, a.scale, a.softcap));
    KC_TRY(fxCache(a.d, Q4, a.v, a.d.v_row, a.d.v_head, "v"));
    if (!aligned(a.out, 4) || !aligned(a.lse, 4) || !aligned(a.part, 4)) return invalid("flash_ext: 4-byte aligned arrays");
    KC_TRY(checkRange(a.out, f32Bytes(int64_t(a.d.N) * a.d.H * a.d.D), "out"));
    if (a.lse) KC_TRY(checkRange(a.lse, f32Bytes(int64_t(a.d.N) * a.d.H), "lse"));
    return checkRange(a.part, f32Bytes(kcamd::fxPlan(a.d).partFloats), "part");
}
template <bool Q4>
int flashExtLaunch(const void* p, void* s) {
    return kcamd::launchFlashExt(Q4, *static_cast<const kcFlashExtArgs*>(p), hs(s));
}

template <bool Q4>
int attnWeightsValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcAttnWeightsArgs*>(p);
    KC_TRY(fxInputs(a.d, Q4, a.q, a.k, a.mask, a.qpos, a.kpos, a.qdoc, a.kdoc, a.slopes, a.scale, a.softcap));
    if (a.w_row < a.d.T) return invalid("attn_weights: w_row holds T values");
    if (!(a.decay == a.decay)) return invalid("attn_weights: decay is a number");
    if (!aligned(a.lse, 4) || !aligned(a.w, 4) || !aligned(a.w_in, 4)) return invalid("attn_weights: 4-byte aligned arrays");
    const size_t w = a.d.T ? (size_t(a.d.H_kv - 1) * size_t(a.w_row) + size_t(a.d.T)) * 4 : 0;
    KC_TRY(checkRange(a.lse, f32Bytes(int64_t(a.d.N) * a.d.H), "lse"));
    if (a.w_in) KC_TRY(checkRange(a.w_in, w, "w_in"));
    return checkRange(a.w, w, "w");
}
template <bool Q4>
int attnWeightsLaunch(const void* p, void* s) {
    return kcamd::launchAttnWeights(Q4, *static_cast<const kcAttnWeightsArgs*>(p), hs(s));
}

int kvKeepValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcKvKeepArgs*>(p);
    if (a.heads <= 0 || a.T < 0 || a.T > INT32_MAX - 2048 || a.w_row < a.T || a.first < 0 || a.recent < 0 || a.n_keep > a.T ||
        int64_t(a.first) + a.recent > a.n_keep || a.keep_row < a.n_keep)
        return invalid("kv_keep: heads positive, first + recent <= n_keep <= T, rows that hold T weights and n_keep positions");
    if (!aligned(a.w, 4) || !aligned(a.keep, 4)) return invalid("kv_keep: 4-byte aligned arrays");
    if (a.T) KC_TRY(checkRange(a.w, (size_t(a.heads - 1) * size_t(a.w_row) + size_t(a.T)) * 4, "w"));
    return checkRange(a.keep, a.n_keep ? (size_t(a.heads - 1) * size_t(a.keep_row) + size_t(a.n_keep)) * 4 : 0, "keep");
}
int kvKeepLaunch(const void* p, void* s) { return kcamd::launchKvKeep(*static_cast<const kcKvKeepArgs*>(p), hs(s)); }

int kvGatherValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcKvGatherArgs*>(p);
    if (a.n_planes < 1 || a.n_planes > 4 || a.heads <= 0 || a.heads > 65535 || a.n_keep < 0 || a.T < 0 || a.keep_row < a.n_keep)
        return invalid("kv_gather: 1 to 4 planes, heads positive, keep_row at least n_keep");
    if (!aligned(a.keep, 4)) return invalid("kv_gather: 4-byte aligned keep");
    if (a.n_keep == 0) return 0;
    KC_TRY(checkRange(a.keep, (size_t(a.heads - 1) * size_t(a.keep_row) + size_t(a.n_keep)) * 4, "keep"));
    int64_t src[4], dst[4];
    for (int i = 0; i < a.n_planes; ++i) {
        const kcKvPlane& q = a.planes[i];
        int64_t s, d;
        if (q.bytes <= 0 || q.bytes % 2 || q.src_row % 2 || q.src_head % 2 || q.dst_row % 2 || q.dst_head % 2 || !aligned(q.src, 2) ||
            !aligned(q.dst, 2) || q.src_row < q.bytes || q.dst_row < q.bytes || q.src_head < 0 || q.dst_head < 0 ||
            (a.heads > 1 && q.dst_head < q.bytes) ||
            !extent(a.heads, q.src_head, q.bytes, &s) || !extent(a.T, q.src_row, s, &src[i]) || !extent(a.heads, q.dst_head, q.bytes, &d) ||
            !extent(a.n_keep, q.dst_row, d, &dst[i]))
            return invalid("kv_gather: bytes and strides even, rows of at least `bytes` bytes");
        KC_TRY(checkRange(q.src, size_t(src[i]), "src"));
        KC_TRY(checkRange(q.dst, size_t(dst[i]), "dst"));
    }
    for (int i = 0; i < a.n_planes; ++i)
        for (int j = 0; j < a.n_planes; ++j) {
            const auto s = reinterpret_cast<uintptr_t>(a.planes[i].src), d = reinterpret_cast<uintptr_t>(a.planes[j].dst);
            if (s < d + uintptr_t(dst[j]) && d < s + uintptr_t(src[i])) return invalid("kv_gather: a destination overlaps a source");
        }
    return 0;
}
int kvGatherLaunch(const void* p, void* s) { return kcamd::launchKvGather(*static_cast<const kcKvGatherArgs*>(p), hs(s)); }

// ---- a step of many requests over a paged cache: kv_pages, rope_ext, flash_pages_f16, sample_rows

bool pageSize(int p) { return p >= 16 && p <= 65536 && (p & (p - 1)) == 0; }
// n ints (or nothing) at 4-byte alignment
int intsAt(const void* p, int64_t n, const char* what) {
    if (!aligned(p, 4)) return invalid("4-byte aligned arrays");
    return checkRange(p, size_t(n) * 4, what);
}
struct Span {
    uintptr_t at;
    size_t bytes;
};
bool overlap(const Span& a, const Span& b) { return a.bytes && b.bytes && a.at < b.at + b.bytes && b.at < a.at + a.bytes; }
Span spanOf(const void* p, size_t bytes) { return {reinterpret_cast<uintptr_t>(p), p ? bytes : 0}; }
// The first `outs` of n arrays overlap neither each other nor the rest.
int apart(const Span* all, int outs, int n, const char* what) {
    for (int i = 0; i < outs; ++i)
        for (int j = i + 1; j < n; ++j)
            if (overlap(all[i], all[j])) return invalid(what);
    return 0;
}

int kvPagesValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcKvPagesArgs*>(p);
    // (each 256 tokens sum over the sequences before them: the limits bound a launch's time)
    if (a.seqs < 0 || a.seqs > (1 << 24) || a.n_tokens < 0 || a.n_tokens > (1 << 24) || a.n_free < 0 || !pageSize(a.page) || a.max_pages < 0 ||
        a.table_row < a.max_pages)
        return invalid("kv_pages: seqs and n_tokens from 0 to 2^24, n_free not negative, page a power of two from 16 to 65536, table_row at least max_pages");
    if ((a.parent != nullptr) != (a.tree != nullptr) || (a.tree ? a.tree_words < 1 || a.tree_words > 64 : a.tree_words != 0))
        return invalid("kv_pages: parent and tree are both given, with 1 to 64 tree_words, or both null, with none");
    if (!aligned(a.slots, 8)) return invalid("kv_pages: slots 8-byte aligned");
    int64_t table;
    if (!extent(a.seqs, int64_t(a.table_row) * 4, int64_t(a.max_pages) * 4, &table)) return invalid("kv_pages: table too large");
    KC_TRY(intsAt(a.have, a.seqs, "have"));
    KC_TRY(intsAt(a.add, a.seqs, "add"));
    KC_TRY(intsAt(a.free, a.n_free, "free"));
    KC_TRY(intsAt(a.table, table / 4, "table"));
    KC_TRY(intsAt(a.start, int64_t(a.seqs) + 1, "start"));
    KC_TRY(intsAt(a.len, a.seqs, "len"));
    KC_TRY(intsAt(a.slots, int64_t(a.n_tokens) * 2, "slots"));
    if (a.pos) KC_TRY(intsAt(a.pos, a.n_tokens, "pos"));
    KC_TRY(intsAt(a.used, 1, "used"));
    if (a.parent) {
        KC_TRY(intsAt(a.parent, a.n_tokens, "parent"));
        KC_TRY(intsAt(a.tree, int64_t(a.n_tokens) * a.tree_words, "tree"));
    }
    const size_t n = size_t(a.n_tokens), s = size_t(a.seqs);
    const Span all[11] = {spanOf(a.table, size_t(table)), spanOf(a.start, 4 * s + 4), spanOf(a.len, 4 * s), spanOf(a.slots, 8 * n), spanOf(a.pos, 4 * n),
                          spanOf(a.used, 4), spanOf(a.tree, 4 * n * size_t(a.tree_words)), spanOf(a.have, 4 * s), spanOf(a.add, 4 * s),
                          spanOf(a.free, 4 * size_t(a.n_free)), spanOf(a.parent, 4 * n)};
    return apart(all, 7, 11, "kv_pages: an output overlaps another array");
}
int kvPagesLaunch(const void* p, void* s) { return kcamd::launchKvPages(*static_cast<const kcKvPagesArgs*>(p), hs(s)); }

// n rows of `heads` heads of `bytes` bytes each, strides in bytes (that of a single row or head is 0).
struct HeadRows {
    Span span;
    int64_t row, head, rowBytes, headBytes, bytes;  // bytes from the first to the last of a row's heads, and of a head's rows
};
HeadRows headRowsOf(const void* p, int64_t n, int64_t row, int64_t heads, int64_t head, int64_t bytes) {  // (after extent: no overflow)
    if (n <= 0 || heads <= 0) return {};
    if (n == 1) row = 0;
    if (heads == 1) head = 0;
    const int64_t x = (heads - 1) * head + bytes, y = (n - 1) * row + bytes;
    return {spanOf(p, p ? size_t(y + x - bytes) : 0), row, head, x, y, bytes};
}
// Whether two such arrays may share a value: not if one ends before the other begins, or if their rows, their heads or all of their values
// repeat at a common distance and lie in different parts of it (q, k and v of a token side by side, K and V in one cache row).
bool mayShare(const HeadRows& a, const HeadRows& b) {
    if (!overlap(a.span, b.span)) return false;
    const auto beside = [&](int64_t step, int64_t x, int64_t y) {
        if (step == 0) return false;
        const int64_t d = a.span.at <= b.span.at ? int64_t(b.span.at - a.span.at) % step : (step - int64_t(a.span.at - b.span.at) % step) % step;
        return d >= x && y <= step - d;
    };
    const int64_t rows = std::gcd(a.row, b.row), heads = std::gcd(a.head, b.head);
    return !beside(rows, a.rowBytes, b.rowBytes) && !beside(heads, a.headBytes, b.headBytes) && !beside(std::gcd(rows, heads), a.bytes, b.bytes);
}
// Rows of `heads` heads of D values, strides in units of `unit` bytes.
int headRows(const void* p, int64_t n, int64_t row, int heads, int64_t head, int D, int unit, const char* what, HeadRows* rows) {
    int64_t x, y;
    if (row < 0 || head < 0 || !aligned(p, size_t(unit)) || !extent(heads, head, D, &x) || !extent(n, row, x, &y) || y > INT64_MAX / 8)
        return invalid("rope_ext: strides not negative, arrays aligned to their values");
    *rows = headRowsOf(p, n, row * unit, heads, head * unit, int64_t(D) * unit);
    return checkRange(p, size_t(y) * size_t(unit), what);
}
// Whether no two of n x heads rows share a value: heads within a row, or rows within a head. (After headRows or extent: no overflow.)
bool rowsApart(int64_t n, int64_t row, int64_t heads, int64_t head, int64_t size) {
    const bool inner = (heads <= 1 || head >= size) && (n <= 1 || row >= (heads - 1) * head + size);
    const bool outer = (n <= 1 || row >= size) && (heads <= 1 || head >= (n - 1) * row + size);
    return inner || outer;
}
int ropeExtValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcRopeExtArgs*>(p);
    if (a.n_tokens < 0 || a.n_tokens > (1 << 29) || a.D <= 0 || a.D % 2 || a.D > 1024 || a.n_rot <= 0 || a.n_rot % 2 || a.n_rot > a.D ||
        (a.interleaved != 0 && a.interleaved != 1))
        return invalid("rope_ext: D even, at most 1024, n_rot even, from 2 to D, interleaved 0 or 1");
    if ((a.q != nullptr) != (a.q_out != nullptr) || (a.k != nullptr) != (a.k_cache != nullptr) || (a.v != nullptr) != (a.v_cache != nullptr) || (a.v && !a.k))
        return invalid("rope_ext: q with q_out, k with k_cache, v with v_cache, and v only with k");
    if (!(a.scale - a.scale == 0.0f)) return invalid("rope_ext: scale is finite");
    if (!aligned(a.freqs, 8) || !aligned(a.slots, 8)) return invalid("rope_ext: freqs and slots 8-byte aligned");
    KC_TRY(intsAt(a.pos, a.n_tokens, "pos"));
    KC_TRY(checkRange(a.freqs, size_t(a.n_rot / 2) * 8, "freqs"));
    HeadRows in[3]{}, out[3]{};
    if (a.q) {
        if (a.H <= 0 || a.H > 65536) return invalid("rope_ext: H from 1 to 65536");
        KC_TRY(headRows(a.q, a.n_tokens, a.q_tok, a.H, a.q_head, a.D, 4, "q", &in[0]));
        KC_TRY(headRows(a.q_out, a.n_tokens, a.out_tok, a.H, a.out_head, a.D, 4, "q_out", &out[0]));
        if (!rowsApart(a.n_tokens, a.out_tok, a.H, a.out_head, a.D)) return invalid("rope_ext: rows of q_out overlap");
    }
    if (a.k) {
        if (a.H_kv <= 0 || a.H_kv > 65536 || a.cache_rows < 0) return invalid("rope_ext: H_kv from 1 to 65536, cache_rows not negative");
        KC_TRY(headRows(a.k, a.n_tokens, a.k_tok, a.H_kv, a.k_head, a.D, 4, "k", &in[1]));
        if (a.v) KC_TRY(headRows(a.v, a.n_tokens, a.v_tok, a.H_kv, a.v_head, a.D, 4, "v", &in[2]));
        KC_TRY(checkRange(a.slots, size_t(a.n_tokens) * 8, "slots"));
        for (int i = 0; i < (a.v ? 2 : 1); ++i) {
            const long long row = i ? a.vc_row : a.kc_row, head = i ? a.vc_head : a.kc_head;
            const int64_t bytes = 2 * int64_t(a.D);
            void* c = i ? a.v_cache : a.k_cache;
            int64_t x, y;
            if (row % 2 || head % 2 || row < 0 || head < 0 || !aligned(c, 2) || !extent(a.H_kv, head, bytes, &x) || !extent(a.cache_rows, row, x, &y))
                return invalid("rope_ext: cache rows, heads and bases at multiples of 2 bytes");
            if (!rowsApart(a.cache_rows, row, a.H_kv, head, bytes)) return invalid("rope_ext: cache rows overlap");
            KC_TRY(checkRange(c, size_t(y), i ? "v_cache" : "k_cache"));
            out[1 + i] = headRowsOf(c, a.cache_rows, row, a.H_kv, head, bytes);
        }
    }
    const Span small[3] = {spanOf(a.pos, size_t(a.n_tokens) * 4), spanOf(a.freqs, size_t(a.n_rot / 2) * 8), spanOf(a.k ? a.slots : nullptr, size_t(a.n_tokens) * 8)};
    const bool inPlace = a.q && a.q_out == a.q && a.out_tok == a.q_tok && a.out_head == a.q_head;
    for (int i = 0; i < 3; ++i)
        for (int j = 0; j < 3; ++j) {
            if (overlap(out[i].span, small[j]) || (i < j && mayShare(out[i], out[j])) || (mayShare(out[i], in[j]) && !(i == 0 && j == 0 && inPlace)))
                return invalid("rope_ext: an output overlaps another array");
        }
    return 0;
}
int ropeExtLaunch(const void* p, void* s) { return kcamd::launchRopeExt(*static_cast<const kcRopeExtArgs*>(p), hs(s)); }

// The sizes alone: what kcFlashPagesPartBytes accepts too.
int fpShape(const kcFlashPagesDims& d) {
    if (d.H <= 0 || d.H_kv <= 0 || d.H % d.H_kv || d.H_kv > 65535 || (d.D != 64 && d.D != 128 && d.D != 256) || d.N < 0 || d.seqs < 0 || d.max_pages < 0 ||
        d.n_pages < 0 || !pageSize(d.page))
        return invalid("flash_pages: H a positive multiple of H_kv, D 64, 128 or 256, counts not negative, page a power of two from 16 to 65536");
    if (int64_t(d.max_pages) * d.page > INT32_MAX - 65536 || d.table_row < d.max_pages)
        return invalid("flash_pages: a sequence's pages hold less than 2^31 - 65536 positions, table_row at least max_pages");
    if (int64_t(d.n_pages) * d.page > INT32_MAX) return invalid("flash_pages: the cache holds less than 2^31 positions");
    if (d.tree_words < 0 || d.tree_words > 64) return invalid("flash_pages: tree_words from 0 to 64");
    if (d.q_tok < 0 || d.q_head < 0 || d.k_row < 0 || d.k_head < 0 || d.v_row < 0 || d.v_head < 0) return invalid("flash_pages: negative strides");
    const int64_t G = d.H / d.H_kv;
    if (int64_t(d.N) * d.H * d.D > INT32_MAX || (int64_t(d.N) * G / 16 + d.seqs) * d.H_kv >= (1 << 24))  // (256 threads for each, below 2^32)
        return invalid("flash_pages: N H D below 2^31, (N H / H_kv / 16 + seqs) H_kv below 2^24");
    return 0;
}
int fpCache(const kcFlashPagesDims& d, const void* p, int64_t row, int64_t head, const char* what, Span* span) {
    int64_t a, b;
    if (row % 16 || head % 16 || !aligned(p, 16)) return invalid("flash_pages: cache rows, heads and base at multiples of 16 bytes");
    if (!extent(d.H_kv, head, int64_t(d.D) * 2, &a) || !extent(int64_t(d.n_pages) * d.page, row, a, &b) || row > INT32_MAX / d.page)
        return invalid("flash_pages: strides too large");
    *span = spanOf(p, size_t(b));
    return checkRange(p, size_t(b), what);
}
int flashPagesValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcFlashPagesArgs*>(p);
    const kcFlashPagesDims& d = a.d;
    KC_TRY(fpShape(d));
    if (!(a.scale - a.scale == 0.0f)) return invalid("flash_pages: scale finite");
    if (a.tree ? d.tree_words < 1 : d.tree_words != 0) return invalid("flash_pages: tree with tree_words, or neither");
    if (!aligned(a.q, 4) || !aligned(a.out, 4) || !aligned(a.lse, 4) || !aligned(a.part, 16)) return invalid("flash_pages: 4-byte aligned arrays, part 16-byte");
    int64_t x, y, t;
    if (!extent(d.H, d.q_head, d.D, &x) || !extent(d.N, d.q_tok, x, &y)) return invalid("flash_pages: q strides too large");
    if (!extent(d.seqs, int64_t(d.table_row) * 4, int64_t(d.max_pages) * 4, &t)) return invalid("flash_pages: table too large");
    KC_TRY(checkRange(a.q, size_t(y) * 4, "q"));
    Span k, v;
    KC_TRY(fpCache(d, a.k, d.k_row, d.k_head, "k", &k));
    KC_TRY(fpCache(d, a.v, d.v_row, d.v_head, "v", &v));
    KC_TRY(intsAt(a.table, t / 4, "table"));
    KC_TRY(intsAt(a.start, d.seqs ? int64_t(d.seqs) + 1 : 0, "start"));
    KC_TRY(intsAt(a.len, d.seqs, "len"));
    if (a.tree) KC_TRY(intsAt(a.tree, int64_t(d.N) * d.tree_words, "tree"));
    KC_TRY(checkRange(a.out, f32Bytes(int64_t(d.N) * d.H * d.D), "out"));
    if (a.lse) KC_TRY(checkRange(a.lse, f32Bytes(int64_t(d.N) * d.H), "lse"));
    const size_t part = kcamd::flashPagesPartBytes(d), n = size_t(d.N), s = size_t(d.seqs);
    KC_TRY(checkRange(a.part, part, "part"));
    const Span all[10] = {spanOf(a.out, 4 * n * size_t(d.H) * size_t(d.D)), spanOf(a.lse, 4 * n * size_t(d.H)), spanOf(a.part, part),
                          spanOf(a.q, size_t(y) * 4), k, v, spanOf(a.table, size_t(t)), spanOf(a.start, s ? 4 * s + 4 : 0), spanOf(a.len, 4 * s),
                          spanOf(a.tree, 4 * n * size_t(d.tree_words))};
    return apart(all, 3, 10, "flash_pages: an output or the workspace overlaps another array");
}
int flashPagesLaunch(const void* p, void* s) { return kcamd::launchFlashPages(*static_cast<const kcFlashPagesArgs*>(p), hs(s)); }

int sampleRowsValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcSampleRowsArgs*>(p);
    int64_t x;
    if (a.rows < 0 || a.rows > 65535 || a.n_vocab <= 0 || a.n_vocab > (1 << 20) || a.row < 0 || !extent(a.rows, a.row, a.n_vocab, &x))
        return invalid("sample_rows: rows from 0 to 65535, n_vocab from 1 to 2^20, row not negative");
    if (!aligned(a.part, 16)) return invalid("sample_rows: part 16-byte aligned");
    if (!aligned(a.logits, 4)) return invalid("sample_rows: 4-byte aligned arrays");
    KC_TRY(checkRange(a.logits, size_t(x) * 4, "logits"));
    KC_TRY(intsAt(a.u, a.rows, "u"));
    if (a.temperature) KC_TRY(intsAt(a.temperature, a.rows, "temperature"));
    if (a.top_k) KC_TRY(intsAt(a.top_k, a.rows, "top_k"));
    if (a.top_p) KC_TRY(intsAt(a.top_p, a.rows, "top_p"));
    if (a.min_p) KC_TRY(intsAt(a.min_p, a.rows, "min_p"));
    KC_TRY(intsAt(a.tokens, a.rows, "tokens"));
    if (a.probs) KC_TRY(intsAt(a.probs, a.rows, "probs"));
    const size_t part = kcamd::sampleRowsPartBytes(a.rows, a.n_vocab), n = 4 * size_t(a.rows);
    KC_TRY(checkRange(a.part, part, "part"));
    const Span all[9] = {spanOf(a.tokens, n), spanOf(a.probs, n), spanOf(a.part, part), spanOf(a.logits, size_t(x) * 4), spanOf(a.u, n),
                         spanOf(a.temperature, n), spanOf(a.top_k, n), spanOf(a.top_p, n), spanOf(a.min_p, n)};
    return apart(all, 3, 9, "sample_rows: an output or the workspace overlaps another array");
}
int sampleRowsLaunch(const void* p, void* s) { return kcamd::launchSampleRows(*static_cast<const kcSampleRowsArgs*>(p), hs(s)); }

// ---- quantize_kquant / fill_normal_f32 (synthetic weights; no reference kernel)

int quantKquantValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcQuantizeKquantArgs*>(p);
    if (a.qtype != KC_QTYPE_Q4_K && a.qtype != KC_QTYPE_Q6_K) return invalid("qtype must be Q4_K (12) or Q6_K (14)");
    if (a.rows < 0 || a.k <= 0 || a.k % 256 != 0 || !fitsIndex(a.rows, a.k / 256))
        return invalid("rows must be non-negative and k a positive multiple of 256");
    const size_t n = size_t(a.rows) * size_t(a.k);
    KC_TRY(checkRange(a.x, n * sizeof(float), "x"));
    return checkRange(a.blocks, n / 256 * (a.qtype == KC_QTYPE_Q6_K ? kcamd::kQ6kBlock : kcamd::kQ4kBlock), "blocks");
}
int quantKquantLaunch(const void* p, void* s) {
    const auto& a = *static_cast<const kcQuantizeKquantArgs*>(p);
    return kcamd::launchQuantizeKquant(a.qtype == KC_QTYPE_Q6_K, a.x, a.blocks, (long long)a.rows * (a.k / 256), hs(s));
}

int fillNormalValidate(const void* p, const kcLaunchContext*) {
    const auto& a = *static_cast<const kcFillNormalArgs*>(p);
    if (a.n < 0) return invalid("n < 0");
    return checkRange(a.y, size_t(a.n) * sizeof(float), "y");
}
int fillNormalLaunch(const void* p, void* s) {
    const auto& a = *static_cast<const kcFillNormalArgs*>(p);
    return kcamd::launchFillNormal(a.y, a.n, a.seed, a.mean, a.stdev, hs(s));
}

const kcKernelEntry kTable[] = {
    {"vector_add", vectorAddValidate, vectorAddLaunch, 1},
    {"quantize_q8x4", quantValidate, quantLaunch, 1},
    {"quantize_cols", quantColsValidate<32>, quantColsLaunch<32>, 1},
    {"quantize_cols_k", quantColsValidate<256>, quantColsLaunch<256>, 1},
    {"matvec_q4k_q8", kquantValidate<false>, kquantLaunch<false>, 1},
    {"matvec_q6k_q8", kquantValidate<true>, kquantLaunch<true>, 1},
    {"matmul_q4k_q8x4", matmulValidate<false, false>, matmulLaunch<false, false>, 1},
    {"matmul_q4k_q8x8", matmulValidate<false, false>, matmulLaunch<false, false>, 1},
    {"matmul_q6k_q8x4", matmulValidate<true, false>, matmulLaunch<true, false>, 1},
    {"matmul_q6k_q8x8", matmulValidate<true, false>, matmulLaunch<true, false>, 1},
    {"matmul_q4k_q8kx4", matmulValidate<false, true>, matmulLaunch<false, true>, 1},
    {"matmul_q4k_q8kx8", matmulValidate<false, true>, matmulLaunch<false, true>, 1},
    {"matmul_q6k_q8kx4", matmulValidate<true, true>, matmulLaunch<true, true>, 1},
    {"matmul_q6k_q8kx8", matmulValidate<true, true>, matmulLaunch<true, true>, 1},
    {"matmul_f16", matmulF16Validate, matmulF16Launch, 1},
    {"add_sumsq_f", addSumsqValidate, addSumsqLaunch, 1},
    {"sumsq_part", sumsqValidate, sumsqLaunch, 1},
    {"norm_mul_q8_f", normMulValidate<false>, normMulLaunch<false>, 1},
    {"norm_mul_q8k_f", normMulValidate<true>, normMulLaunch<true>, 1},
    {"add_norm_q8_f", addNormValidate, addNormLaunch, 1},
    {"silu_mul_q8x4f", siluQValidate<false>, siluQLaunch<false>, 1},
    {"silu_mul_q8kf", siluQValidate<true>, siluQLaunch<true>, 1},
    {"rms_norm", rmsValidate, rmsLaunch, 1},
    {"mul_rows", mulRowsValidate, mulRowsLaunch, 0},
    {"silu_mul", siluValidate, siluLaunch, 1},
    {"rope_ggml", ropeValidate, ropeLaunch, 0},
    {"set_rows_f16", setRowsValidate, setRowsLaunch, 1},
    {"fa_scores", faScoresValidate, faScoresLaunch, 1},
    {"fa_max", faMaxValidate, faMaxLaunch, 1},
    {"fa_exp", faExpValidate, faExpLaunch, 1},
    {"fa_values", faValuesValidate, faValuesLaunch, 1},
    {"flash_attn_f16", flashValidate, flashLaunch, 0},
    {"flash_decode_f16", flashDecodeValidate, flashDecodeLaunch, 0},
    {"set_rows_q4_0", setRowsQ40Validate, setRowsQ40Launch, 0},
    {"get_rows_q4_0", getRowsQ40Validate, getRowsQ40Launch, 0},
    {"flash_ext_f16", flashExtValidate<false>, flashExtLaunch<false>, 0},
    {"flash_ext_q4_0", flashExtValidate<true>, flashExtLaunch<true>, 0},
    {"attn_weights_f16", attnWeightsValidate<false>, attnWeightsLaunch<false>, 0},
    {"attn_weights_q4_0", attnWeightsValidate<true>, attnWeightsLaunch<true>, 0},
    {"kv_keep", kvKeepValidate, kvKeepLaunch, 0},
    {"kv_gather", kvGatherValidate, kvGatherLaunch, 0},
    {"kv_pages", kvPagesValidate, kvPagesLaunch, 0},
    {"rope_ext", ropeExtValidate, ropeExtLaunch, 0},
    {"flash_pages_f16", flashPagesValidate, flashPagesLaunch, 0},
    {"sample_rows", sampleRowsValidate, sampleRowsLaunch, 0},
    {"repack_kquant", repackValidate<false>, repackLaunch<false>, 0},
    {"unpack_kquant", repackValidate<true>, repackLaunch<true>, 0},
    {"get_rows_kquant", getRowsValidate, getRowsLaunch, 0},
    {"quantize_kquant", quantKquantValidate, quantKquantLaunch, 0},
    {"fill_normal_f32", fillNormalValidate, fillNormalLaunch, 0},
};

}  // namespace

const kcKernelEntry* kcamd::builtinKernels(size_t* count) {
    *count = sizeof kTable / sizeof kTable[0];
    return kTable;
}

kcError_t kcKquantStreamBytes(int qtype, int rows, int k, size_t* bytes) noexcept {
    if (!bytes || (qtype != KC_QTYPE_Q4_K && qtype != KC_QTYPE_Q6_K) || rows < 0 || k <= 0 || k % 256 != 0)
        return kc::Error::InvalidValue;
    *bytes = kcamd::streamBytes(qtype == KC_QTYPE_Q6_K, rows, k);
    return kc::Error::Success;
}

kcError_t kcFlashExtPartBytes(const kcFlashExtDims* dims, size_t* bytes) noexcept {
    if (!dims || !bytes || fxShape(*dims)) return kc::Error::InvalidValue;
    *bytes = f32Bytes(kcamd::fxPlan(*dims).partFloats);
    return kc::Error::Success;
}

kcError_t kcFlashPagesPartBytes(const kcFlashPagesDims* dims, size_t* bytes) noexcept {
    if (!dims || !bytes || fpShape(*dims)) return kc::Error::InvalidValue;
    *bytes = kcamd::flashPagesPartBytes(*dims);
    return kc::Error::Success;
}

kcError_t kcSampleRowsPartBytes(int rows, int n_vocab, size_t* bytes) noexcept {
    if (!bytes || rows < 0 || rows > 65535 || n_vocab <= 0 || n_vocab > (1 << 20)) return kc::Error::InvalidValue;
    *bytes = kcamd::sampleRowsPartBytes(rows, n_vocab);
    return kc::Error::Success;
}
