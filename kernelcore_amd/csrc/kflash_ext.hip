// kflash_ext.hip -- flash_ext_f16 / flash_ext_q4_0 (gfx950): attention of N query tokens over T cached positions of an
// fp16 or a 4-bit cache with shaped scores: for query row i of a KV head (kflash_ext_device.hpp packs tokens and the
// group's heads into rows)
//   x_ij = log2 e (cap tanh(scale q_i.k_j / cap) - slope_i |pos_i - pos_j| + mask_ij),   o_i = sum_j 2^(x_ij - m_i) v_j / l_i,
//   m_i = max_j x_ij, l_i = sum_j 2^(x_ij - m_i)
// over the keys that i sees, in one pass over the keys with running m and l.
//
// Three kernels: few rows (single and drafted tokens, short calls), many rows (prompts), and the join of key ranges where
// a call's rows alone do not fill the GPU.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "internal.hpp"
#include "kflash_ext_device.hpp"

namespace kcamd {
namespace {

using namespace fx;

// A row's m may lag behind its maximum by up to kLag (p = 2^(x - m) up to 16), so that the sums are rescaled rarely; p is split
// into fp16 parts at the scale 2^11 (up to 2^15 then), so that what the parts cannot hold is below 2^-36 of the largest p.
// (x - m + 11 is what is exponentiated; l and o carry the factor until the end.)
constexpr float kLag = 4.0f, kPBits = 11.0f, kPInv = 1.0f / 2048.0f;

// Row r of a workgroup's range, whose sums came out NaN, from the definition: written as the kernels write their rows, by a wavefront.
template <int D, bool Q4, int TK>
__device__ __forceinline__ void writePlainRow(int kvh, int r, int sp, int lane) {
    const FxParams a = paramsAgain();
    float m, l, o[D / 64];
    plainRow<D, Q4, TK>(a, kvh, r, sp, lane, m, l, o);
    const int token = r / a.G, head = kvh * a.G + (r - token * a.G);
    const size_t at = ((size_t)sp * a.H_kv + kvh) * a.rows + r;
    const bool whole = a.splits == 1;
    float* dst = whole ? a.out + ((size_t)token * a.H + head) * D : a.part + at * D;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) dst[lane + 64 * e] = !whole ? o[e] : l == 0.0f ? 0.0f : o[e] / l;
    if (lane) return;
    if (!whole) {
        float* ml = a.part + (size_t)a.splits * a.H_kv * a.rows * D + 2 * at;
        ml[0] = m;
        ml[1] = l;
    } else if (a.lse) {
        a.lse[(size_t)token * a.H + head] = l == 0.0f ? -INFINITY : fmaf(m, kLn2, logf(l));
    }
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
// A word's infinities and NaNs as zeros.
__device__ __forceinline__ uint32_t tameHalves(uint32_t w) {
    const uint32_t z = wildHalves(w);
    return w & ~((z >> 15 & 1u) * 0xFFFFu | (z >> 31) * 0xFFFF0000u);
}

// ---------------------------------------------------------------------------------------------- many rows
// Workgroup: 128 rows of a KV head (four wavefronts of 32 rows) over one range of keys. A step takes KS tiles of 32 keys; with
// KS = 2 two sets of four wavefronts take a tile each, joined through LDS at the end. Matrix form (v_mfma_f32_32x32x16_f16,
// lane (j, h) = row j, lane half h):
//   S^T = K Q^T: A = key rows (LDS), B = q hi / lo (registers). Lane (j, h) holds keys 8 (v / 4) + 4 h + v % 4 of row j.
//   O^T += V^T P^T: A = V^T through transposed LDS reads, B = p hi / lo, the score registers as they are (the products'
//   index runs over the keys in the order those registers hold).
// 4-bit keys and values are unpacked once per workgroup, on the way to LDS (by each wavefront, after reads of the codes: 176
// against 165 us for 1000 tokens over 3577 positions); a step's keys and values lie in one of two
// buffers, the next step's stored while the present one is computed and the loads of the one after in flight, one barrier a step. The
// two wavefronts of a SIMD drift apart within a step, and one's softmax runs beside the other's products. (Keeping them half
// a step apart by a second barrier, the values' products a step behind, was slower: 103 against 94 us for 2048 tokens. So was one
// set to a workgroup: 101 against 78 us.)
// Bound by the products, staging and softmax, which overlap little: 2048 causal tokens, 24 heads of 128, fp16: 75 us, 0.69
// PFLOP/s counting both parts of q and p (a large fp16 product of the library: 1.19); 1000 tokens over 3577 4-bit positions,
// 32 heads: 147 us, 0.86 PFLOP/s.
template <int D, bool Q4>
struct Geo {
    static constexpr int KS = D == 256 ? 1 : 2;  // (256 values: one wavefront's registers fill a SIMD)
    static constexpr int Threads = 256 * KS, TK = 32 * KS;
    static constexpr int NB = D / 32;
    static constexpr int KRow = kKeyRow<D>;
    static constexpr int VRow = 2 * D + 32;  // two pad chunks, for the transposed reads
    static constexpr int oScale = TK * KRow;                              // 4-bit: the keys' scales
    static constexpr int oV = oScale + (Q4 ? NB * TK * 2 : 0), oLow = TK * VRow;  // values, 4-bit: their rests
    static constexpr int oMeta = oV + TK * VRow * (Q4 ? 2 : 1);           // positions, document numbers
    static constexpr int QRow = 2 * D + 16;                           // a row of q: fp16 values hi, their lo parts
    static constexpr int Buf = oMeta + TK * 8, oMap = 2 * Buf > 256 * QRow ? 2 * Buf : 256 * QRow;
    static constexpr int MapEntries = 2048;      // 256 keys each: the steps with a key that some row may see, those all rows see
    static constexpr int oWild = oMap + 2 * MapEntries;  // 3 x the step's wild keys
    static constexpr int oZ = oWild + 32;                // a wild key's values, for each wavefront
    static constexpr int oTops = oZ;                     // and, before the first step, the rows' largest |q|
    static constexpr int OV = D / 16;            // the join of the two sets: vectors of four per lane
    static constexpr int Join = KS == 2 ? 512 * (OV * 16 + 8) : 0;
    static constexpr int End = oZ + 4 * KS * D * 4;
    static constexpr int Lds = End > Join ? End : Join;
};

template <int D, bool Q4, bool SHAPED>
__global__ __launch_bounds__(256 * (D == 256 ? 1 : 2), D == 256 ? 1 : 2) void flash_ext_kernel(FxParams a) {
    using G = Geo<D, Q4>;
    constexpr int DB = D / 32, NB = G::NB, TK = G::TK, NT = G::Threads, SPC = 256 / TK;
    extern __shared__ int4 lds4[];
    char* lds = reinterpret_cast<char*>(lds4);
    unsigned short* map = reinterpret_cast<unsigned short*>(lds + G::oMap);
    int* wildAt = reinterpret_cast<int*>(lds + G::oWild);
    const int kvh = blockIdx.x, rb = (int)gridDim.y - 1 - (int)blockIdx.y, sp = blockIdx.z;  // (longest rows first)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j = lane & 31, h = lane >> 5, rw = wave & 3, ks = wave >> 2;
    const int r0 = rb * 128 + rw * 32, r = r0 + j;
    const Row row = rowOf(a, kvh, r);
    RowQ<D / G::KS> q;  // (each set takes its part of the values)
    q.load(a.q + ks * (D / G::KS), (long long)row.token * a.q_tok + (long long)row.head * a.q_head, lane);
    const unsigned short* mrow = SHAPED && a.mask ? a.mask + (size_t)row.token * a.m_row2 : nullptr;
    const bool meta = SHAPED && (a.kpos || a.kdoc);
    const int* kpos = SHAPED && a.kpos ? a.kpos + (size_t)kvh * a.key_row : nullptr;
    const int* kdoc = SHAPED && a.kdoc ? a.kdoc + (size_t)kvh * a.key_row : nullptr;

    // the least and largest position limit of the wavefront's rows and of the workgroup's, and of their document numbers
    int wmin, wmax, bmin, bmax, dmin = 0, dmax = 0;
    const int b0 = rb * 128 / a.G, b1 = min(rb * 128 + 127, a.rows - 1) / a.G;  // the workgroup's tokens
    if (!(SHAPED && a.qpos)) {  // (ascending with the rows)
        wmin = r0 < a.rows ? limitOf(a, a.pos0 + r0 / a.G) : INT_MAX;
        wmax = r0 < a.rows ? limitOf(a, a.pos0 + min(r0 + 31, a.rows - 1) / a.G) : -1;
        bmin = limitOf(a, a.pos0 + b0);
        bmax = limitOf(a, a.pos0 + b1);
    } else {
        wmin = waveMin(row.live ? row.limit : INT_MAX);
        wmax = waveMax(row.live ? row.limit : -1);
        const int l0 = limitOf(a, a.qpos[min(b0 + lane, b1)]), l1 = limitOf(a, a.qpos[min(b0 + 64 + lane, b1)]);
        bmin = waveMin(min(l0, l1));
        bmax = waveMax(max(l0, l1));
    }

    // this range's steps, every splits-th of all (what the rows see is spread over the ranges): step i of the range is step
    // stepOf(i); the range's end before i1
    int t1 = a.T / TK + (a.T % TK != 0);
    if (!kpos) t1 = bmax < 0 ? 0 : min(t1, bmax / TK + 1);
    const int i1 = t1 > sp ? (t1 - sp + a.splits - 1) / a.splits : 0, chunks = (i1 + SPC - 1) / SPC;
    auto stepOf = [&](int i) { return i * a.splits + sp; };
    const bool mapped = meta && chunks <= G::MapEntries;
    if constexpr (SHAPED) {
        if (mapped) {  // a wavefront takes 256 keys, four a lane
            constexpr int LPT = TK / 4;  // lanes to a step
            const int key1 = min(a.T, t1 * TK), n = chunks;
            int p[4], x[4];
            auto keysOf = [&](int at) {
                const int key = stepOf(at * SPC + lane / LPT) * TK + 4 * (lane % LPT);
                if (key + 3 < key1) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = key + e;
                    if (kpos) *reinterpret_cast<int4*>(p) = *reinterpret_cast<const int4a4*>(kpos + key);
                    if (kdoc) *reinterpret_cast<int4*>(x) = *reinterpret_cast<const int4a4*>(kdoc + key);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[e] = key + e >= key1 ? -1 : kpos ? kpos[key + e] : key + e;
                        x[e] = kdoc && key + e < key1 ? kdoc[key + e] : 0;
                    }
                }
            };
            int at = wave;
            if (at < n) keysOf(at);
            if (a.qdoc) {
                const int d0 = a.qdoc[min(b0 + lane, b1)], d1 = a.qdoc[min(b0 + 64 + lane, b1)];
                dmin = waveMin(min(d0, d1));
                dmax = waveMax(max(d0, d1));
            }
            for (; at < n; at += NT / 64) {
                bool some = false, all = true;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool in = p[e] >= 0 && p[e] <= bmax && (!kdoc || (x[e] >= dmin && x[e] <= dmax));
                    some |= in;
                    all &= in && p[e] <= bmin && dmin == dmax;
                }
                const unsigned long long s = __ballot(some), w = __ballot(all), group = (1ull << LPT) - 1;
                const unsigned long long sb = __ballot(lane < SPC && (s >> (lane % SPC * LPT) & group)),
                                         wb = __ballot(lane < SPC && (w >> (lane % SPC * LPT) & group) == group);
                if (lane == 0) map[at] = (unsigned short)(sb | wb << 8);
                if (at + NT / 64 < n) keysOf(at + NT / 64);
            }
        }
    }
    float* tops = reinterpret_cast<float*>(lds + G::oTops) + rw * 32;
    q.tops(tops + ks * 128, lane);
    if (tid < 8) wildAt[tid] = 0;
    __syncthreads();
    auto next = [&](int i) -> int {  // the first step from i on that is to be computed; i1 if none
        if (!mapped) return min(i, i1);
        while (i < i1) {
            const uint32_t w = (__builtin_amdgcn_readfirstlane(map[i / SPC]) & 0xFFu) >> (i % SPC);
            if (w) return i + __builtin_ctz(w);
            i = (i / SPC + 1) * SPC;
        }
        return i1;
    };

    // ---- staging, through registers: 16-byte chunks (fp16) or half blocks of 8 bytes (4-bit) of a step's K and V rows, of each NL
    // per thread. Addresses: the step's first row, the same for the workgroup, + the thread's share.
    constexpr int PR = Q4 ? 2 * NB : D / 8, IT = TK * PR, NL = (IT + NT - 1) / NT;
    typedef __attribute__((ext_vector_type(Q4 ? 2 : 4))) uint32_t Item;
    Item kraw[NL], vraw[NL];
    uint32_t ksc[Q4 ? NL : 1], vsc[Q4 ? NL : 1];
    int rmeta = 0;
    const char* kb = a.k + (size_t)kvh * a.k_head;
    const char* vb = a.v + (size_t)kvh * a.v_head;
    const int part = tid % PR, key0 = tid / PR;                       // (NT is a multiple of PR)
    const int pb = Q4 ? 18 * (part >> 1) : 16 * part;                 // the block, or the chunk
    const bool idle = IT < NT && tid >= IT;
    auto load = [&](const char* p, Item& x, uint32_t& sc) {
        if constexpr (Q4) {
            x = *reinterpret_cast<const __attribute__((aligned(2))) Item*>(p + 2 + 8 * (part & 1));
            sc = *reinterpret_cast<const u32a2*>(p);
        } else {
            x = *reinterpret_cast<const __attribute__((aligned(4))) Item*>(p);
        }
    };
    const long long klane = key0 * a.k_row + pb, vlane0 = key0 * a.v_row + pb;
    auto fetch = [&](int t) {
        if (!idle) {
            const char *kt = kb + (long long)t * TK * a.k_row, *vt = vb + (long long)t * TK * a.v_row;
            if (t * TK + TK <= a.T) {
#pragma unroll
                for (int n = 0; n < NL; ++n) {
                    load(kt + NT / PR * n * a.k_row + klane, kraw[n], ksc[Q4 ? n : 0]);
                    load(vt + NT / PR * n * a.v_row + vlane0, vraw[n], vsc[Q4 ? n : 0]);
                }
            } else {
                asm volatile("" ::: "memory");  // (a branch: as selects, its products would be every step's)
#pragma unroll
                for (int n = 0; n < NL; ++n) {  // rows past the end reread the last one
                    const long long at = min(NT / PR * n + key0, a.T - 1 - t * TK);
                    load(kt + at * a.k_row + pb, kraw[n], ksc[Q4 ? n : 0]);
                    load(vt + at * a.v_row + pb, vraw[n], vsc[Q4 ? n : 0]);
                }
            }
        }
        if constexpr (SHAPED) {
            if (meta && tid < 2 * TK) {
                const int key = min(t * TK + tid % TK, a.T - 1);
                const int* src = tid < TK ? kpos : kdoc;
                rmeta = src ? src[key] : tid < TK ? key : 0;
            }
        }
    };
    // (whatever is done to a loaded value is done here: done in fetch, it would wait for the loads there)
    auto store = [&](int t, char* buf, int* wild) {
        if (t * TK + TK > a.T) {  // values past the end are 0
            asm volatile("" ::: "memory");
#pragma unroll
            for (int n = 0; n < NL; ++n)
                if (t * TK + NT / PR * n + key0 >= a.T) {
                    vsc[Q4 ? n : 0] = 0;
                    if constexpr (!Q4) vraw[n] = Item{};
                }
        }
        if (!idle) {
#pragma unroll
            for (int n = 0; n < NL; ++n) {
                const int key = NT / PR * n + key0;
                char* pk = buf + key * G::KRow + (Q4 ? 64 * (part >> 1) + 16 * (part & 1) : 16 * part);
                char* pv = buf + G::oV + key * G::VRow + (Q4 ? 64 * (part >> 1) + 16 * (part & 1) : 16 * part);
                if constexpr (Q4) {
                    h8 lo, hi;  // values 8 (part % 2) .. + 8 of the block, and those 16 on
                    byteCodes8(kraw[n], lo, hi);
                    *reinterpret_cast<h8*>(pk) = lo;
                    *reinterpret_cast<h8*>(pk + 32) = hi;
                    if (!(part & 1))
                        reinterpret_cast<_Float16*>(buf + G::oScale)[(key >> 5) * NB * 32 + scaleAt(part >> 1, key & 31)] =
                            finiteOrNaN(__builtin_bit_cast(_Float16, (unsigned short)ksc[n]));
                    uint32_t s = vsc[n] & 0xFFFFu;
                    if (wildScale(s)) {
                        s = 0;
                        atomicOr(wild + (key >> 5), 1 << (key & 31));
                    }
                    const _Float16 d1 = __builtin_bit_cast(_Float16, (unsigned short)s);
                    const h8 d = {d1, d1, d1, d1, d1, d1, d1, d1};
                    byteCodes8(vraw[n], lo, hi);
                    const h8 x = lo * d, y = hi * d;
                    *reinterpret_cast<h8*>(pv) = x;
                    *reinterpret_cast<h8*>(pv + 32) = y;
                    *reinterpret_cast<h8*>(pv + G::oLow) = __builtin_elementwise_fma(lo, d, -x);
                    *reinterpret_cast<h8*>(pv + G::oLow + 32) = __builtin_elementwise_fma(hi, d, -y);
                } else {
                    *reinterpret_cast<Item*>(pk) = kraw[n];
                    float squares = 0.0f;  // infinite or NaN where one of the values is
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t word = vraw[n][w];  // (a bit cast of the element itself takes the vector's first)
                        const h2 x = __builtin_bit_cast(h2, word);
                        squares = __builtin_amdgcn_fdot2(x, x, squares, false);
                    }
                    if (!(squares < INFINITY)) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) vraw[n][w] = tameHalves(vraw[n][w]);
                        atomicOr(wild + (key >> 5), 1 << (key & 31));
                    }
                    *reinterpret_cast<Item*>(pv) = vraw[n];
                }
            }
        }
        if constexpr (SHAPED)
            if (meta && tid < 2 * TK)
                reinterpret_cast<int*>(buf + G::oMeta)[tid] = tid < TK && (rmeta < 0 || t * TK + tid >= a.T) ? kNoKey : rmeta;
    };

    const Shape shape = SHAPED ? shapeOf(a) : Shape{};
    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    int i = next(0), in = i < i1 ? next(i + 1) : i1;
    if (i < i1) fetch(stepOf(i));
    h8 qh[D / 16], ql[D / 16];
    auto topOf = [&](int r) { return G::KS == 2 ? fmaxf(tops[r], tops[128 + r]) : tops[r]; };
    const float c = qScale(topOf(j), a.scale).c, c2 = factor2(c);
    {
        _Float16* qr = reinterpret_cast<_Float16*>(lds) + rw * 32 * G::QRow;
        h4 low[RowQ<D / G::KS>::N];
        q.split(a, qr + ks * (D / G::KS), G::QRow, lane, topOf, low);
        q.place(qr + D + 8 + ks * (D / G::KS), G::QRow, lane, low);
        __syncthreads();
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
            qh[n] = *reinterpret_cast<const h8*>(qr + j * G::QRow + 16 * n + 8 * h);
            ql[n] = *reinterpret_cast<const h8*>(qr + j * G::QRow + D + 8 + 16 * n + 8 * h);
        }
    }
    __syncthreads();
    if (i < i1) store(stepOf(i), lds, wildAt);
    if (in < i1) fetch(stepOf(in));
    __syncthreads();
    const int vlane = ks * 32 * (G::VRow / 2) + (4 * (lane >> 5) + ((lane & 15) >> 2)) * (G::VRow / 2) + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    int slot = 0;  // of the wild-key words: three pairs in turn, the one two steps on is cleared while none reads it
    for (int it = 0; i < i1; ++it) {
        const int t = stepOf(i);
        char* cur = lds + (it & 1) * G::Buf;
        const int sn = slot == 2 ? 0 : slot + 1, sc = sn == 2 ? 0 : sn + 1, inn = in < i1 ? next(in + 1) : i1;
        const int k0 = t * TK + 32 * ks;  // this wavefront's 32 keys
        bool full = !(SHAPED && mrow) && k0 + 31 < a.T;
        if (meta) full = full && mapped && (__builtin_amdgcn_readfirstlane(map[i / SPC]) >> (8 + i % SPC) & 1);
        else full = full && k0 + 31 <= wmin;
        const bool work = full || meta || k0 <= wmax;
        // the next step into the other buffer (last read before the barrier that ended the step before this one): the second set
        // now, beside the first one's products, the first set at the end, beside the second one's
        auto stage = [&]() {
            if (in < i1) store(stepOf(in), lds + ((it + 1) & 1) * G::Buf, wildAt + 2 * sn);
            if (inn < i1) fetch(stepOf(inn));
        };
        MaskWords mk;
        if constexpr (SHAPED) {
            if (mrow && work) mk.load(mrow, t * (TK / 32) + ks, h, a.T);
        }
        if (ks == 1) stage();
        float x[16];
        if (work) keyScores<D, Q4>(cur + ks * 32 * G::KRow, cur + G::oScale + ks * NB * 64, j, h, qh, ql, x);
        if (work) {
            const int wildBits = wildAt[2 * slot + ks];
            const int* kp = reinterpret_cast<const int*>(cur + G::oMeta) + 32 * ks + 4 * h;
            if constexpr (SHAPED) shapeScores(x, c, shape, row, meta ? kp : nullptr, k0 + 4 * h, mrow != nullptr, mk);
            if (!full) {
                if (meta) {
                    hideKeys(x, row, kp, kp + TK);
                } else {
                    const int last = min(row.limit, a.T - 1) - k0 - 4 * h;
#pragma unroll
                    for (int v = 0; v < 16; ++v) x[v] = 8 * (v >> 2) + (v & 3) <= last ? x[v] : -INFINITY;
                }
            }
            float bm = x[0];
#pragma unroll
            for (int v = 1; v < 16; ++v) bm = fmaxf(bm, x[v]);
            bm = swap32Max(bm);
            if constexpr (!SHAPED) bm *= c2;
            // a row's m follows its maximum only when that is more than kLag ahead: after the first keys hardly ever
            const bool ahead = bm > m + kLag;
            if (__any(ahead)) {
                const float mn = ahead ? bm : m, alpha = ahead ? ex2(m - mn) : 1.0f;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int v = 0; v < 16; ++v) o[d][v] *= alpha;
                m = mn;
            }
            const float off = kPBits - (m == -INFINITY ? 0.0f : m);  // (nothing seen yet: every p is 0)
            float ls = 0.0f;
#pragma unroll
            for (int v = 0; v < 16; ++v) {
                x[v] = ex2(SHAPED ? x[v] + off : fmaf(x[v], c2, off));
                ls += x[v];
            }
            l += ls;
            uint32_t wild = __builtin_amdgcn_readfirstlane(wildBits);
            if (__builtin_expect(wild != 0, 0)) {  // values that are no matrix operands, for the rows that see them
                float* zr = reinterpret_cast<float*>(lds + G::oZ) + wave * D;
#pragma unroll 1
                while (wild) {
                    const int key = __builtin_ctz(wild);
                    wild &= wild - 1;
                    const float p = __shfl(pick<16>(x, (key >> 3) * 4 + (key & 3)), j + 32 * ((key >> 2) & 1));
                    if (!__any(p != 0.0f)) continue;
                    const char* vr = vb + (size_t)(k0 + key) * a.v_row;
#pragma unroll
                    for (int e = 0; e < D / 64; ++e) zr[lane + 64 * e] = wildValue<Q4>(vr, lane + 64 * e);
                    waveLds();
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const f32x4 z = *reinterpret_cast<const f32x4*>(zr + 32 * d + 8 * g + 4 * h);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float y = fmaf(p, z[e], o[d][4 * g + e]);
                                o[d][4 * g + e] = p != 0.0f ? y : o[d][4 * g + e];
                            }
                        }
                    waveLds();
                }
            }
            h8 ph[2], pl[2];
            splitParts<16>(x, ph, pl);
            const _Float16* vcol = reinterpret_cast<const _Float16*>(cur + G::oV) + vlane;
#pragma unroll
            for (int mm = 0; mm < 2; ++mm)
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const _Float16* vp = vcol + 16 * mm * (G::VRow / 2) + 32 * d;
                    const s4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)vp);
                    const s4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(vp + 8 * (G::VRow / 2)));
                    const h8 va = __builtin_bit_cast(h8, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, ph[mm], o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, pl[mm], o[d], 0, 0, 0);
                    if constexpr (Q4) {
                        const _Float16* vq = vp + G::oLow / 2;
                        const s4 y0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)vq);
                        const s4 y1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4)(vq + 8 * (G::VRow / 2)));
                        const h8 vl = __builtin_bit_cast(h8, __builtin_shufflevector(y0, y1, 0, 1, 2, 3, 4, 5, 6, 7));
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vl, ph[mm], o[d], 0, 0, 0);
                    }
                }
        }
        if (ks == 0) stage();
        if (tid < 2) wildAt[2 * sc + tid] = 0;
        slot = sn;
        i = in;
        in = inn;
        __syncthreads();
    }

    // the two sets swap halves of their sums, each joins and writes one half of the values
    l += __shfl_xor(l, 32);
    constexpr int OB = DB / G::KS;  // blocks of 32 values that a wavefront writes
    const int d0 = ks * OB;
    if constexpr (G::KS == 2) {
        f32x4* mg = reinterpret_cast<f32x4*>(lds) + (size_t)wave * 64 * G::OV + lane;
        float2* ml = reinterpret_cast<float2*>(lds + 8 * 64 * G::OV * 16) + wave * 64 + lane;
#pragma unroll
        for (int d = 0; d < OB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x16 &u = o[d], &w = o[OB + d];
                mg[64 * (4 * d + g)] = ks ? f32x4{u[4 * g], u[4 * g + 1], u[4 * g + 2], u[4 * g + 3]}
                                          : f32x4{w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]};
            }
        *ml = make_float2(m, l);
        __syncthreads();
        mg += ks ? -4 * 64 * G::OV : 4 * 64 * G::OV;
        ml += ks ? -256 : 256;
        const float m1 = ml->x, l1 = ml->y, M = fmaxf(m, m1);
        const float f0 = m == -INFINITY ? 0.0f : ex2(m - M), f1 = m1 == -INFINITY ? 0.0f : ex2(m1 - M);
        l = ks ? l1 * f1 + l * f0 : l * f0 + l1 * f1;
        m = M;
#pragma unroll
        for (int d = 0; d < OB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 y = mg[64 * (4 * d + g)];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float own = ks ? o[OB + d][4 * g + e] : o[d][4 * g + e];
                    o[d][4 * g + e] = own * f0 + y[e] * f1;
                }
            }
    }
    if (row.live && l == l) {
        float* dst;
        float f;
        if (a.splits == 1) {
            dst = a.out + ((size_t)row.token * a.H + row.head) * D;
            f = l == 0.0f ? 0.0f : 1.0f / l;
            if (a.lse && h == 0 && ks == 0) a.lse[(size_t)row.token * a.H + row.head] = l == 0.0f ? -INFINITY : fmaf(m, kLn2, logf(l * kPInv));
        } else {
            const size_t at = ((size_t)sp * a.H_kv + kvh) * a.rows + r;
            dst = a.part + at * D;
            f = kPInv;
            if (h == 0 && ks == 0) {
                float* ml = a.part + (size_t)a.splits * a.H_kv * a.rows * D + 2 * at;
                ml[0] = m;
                ml[1] = l * kPInv;
            }
        }
#pragma unroll
        for (int d = 0; d < OB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 y = {o[d][4 * g] * f, o[d][4 * g + 1] * f, o[d][4 * g + 2] * f, o[d][4 * g + 3] * f};
                *reinterpret_cast<f4a4*>(dst + 32 * (d0 + d) + 8 * g + 4 * h) = y;
            }
    }
    unsigned again = (unsigned)__ballot(row.live && l != l && (G::KS == 1 || (j & 1) == ks));  // (the sets share them)
    for (; __builtin_expect(again != 0, 0); again &= again - 1) writePlainRow<D, Q4, TK>(kvh, r0 + __builtin_ctz(again), sp, lane);
}

// ---------------------------------------------------------------------------------------------- few rows
// Groups of up to 32 rows (NR columns of 16): single tokens and a few drafted ones, where the cache's bytes count, and more rows over
// short ranges, where latency does (fxPlan). One token of 32 heads over
// 131072 4-bit positions: 47 us, 3.2 TB/s of cache, by its unpacking most of all (770 VALU instructions
// per 64 keys, start and join included, half of the time); over 8191:
// 8.5 us, of which 2 are the first tile's latency and 3 its computation. Workgroup: four
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
    static constexpr int oMeta = Q4 ? oD + NB * 128 : 32 * VRow;  // positions, document numbers
    static constexpr int oZ = oMeta + TK * 8;  // a wild key's values
    static constexpr int Wave = oZ + D * 4;
    static constexpr int ORow = D + 4;       // join: floats per row
    static constexpr int Join = 4 * NR * 16 * (ORow + 2) * 4;
    static constexpr int Lds = 4 * Wave > Join ? 4 * Wave : Join;
};

template <int D, bool Q4, bool SHAPED, int NR>
__global__ __launch_bounds__(256, D == 256 || NR == 2 ? 1 : 2) void flash_ext_few_kernel(FxParams a) {
    using G = FewGeo<D, Q4, NR>;
    constexpr int NB = G::NB, TK = G::TK, U = TK / 16, TT = TK / 32, DT = D / 16;
    extern __shared__ int4 lds4[];
    char* lds = reinterpret_cast<char*>(lds4);
    const int sp = blockIdx.x, kvh = blockIdx.y, row0 = blockIdx.z * 16 * NR, rows = min(a.rows - row0, 16 * NR);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i = lane & 15, kg = lane >> 4;
    char* mine = lds + wave * G::Wave;
    const char* kb = a.k + (size_t)kvh * a.k_head;
    const char* vb = a.v + (size_t)kvh * a.v_head;
    int t1 = a.T / TK + (a.T % TK != 0);

    const bool meta = SHAPED && (a.kpos || a.kdoc);
    const int* kpos = SHAPED && a.kpos ? a.kpos + (size_t)kvh * a.key_row : nullptr;
    const int* kdoc = SHAPED && a.kdoc ? a.kdoc + (size_t)kvh * a.key_row : nullptr;

    // a tile's loads. 4-bit: blocks lane + 64 n of the tile's 64 NB. fp16: K as the A operand [u][b], V chunks lane + 64 n.
    // Addresses: the tile's first row (the same for the wavefront) + the lane's share; rows past the end reread the last one.
    constexpr int NV = Q4 ? NB : 2 * NB, PR = Q4 ? NB : D / 8;  // V items per lane; items of a row
    u4 kr[NV], vr[NV];
    uint32_t kscale[Q4 ? NB : 1], vscale[Q4 ? NB : 1];
    const long long klane = Q4 ? (long long)(lane / PR) * a.k_row + 18 * (lane % PR) : (long long)i * a.k_row + 16 * kg;
    const long long vlane = (long long)(lane / PR) * a.v_row + (Q4 ? 18 : 16) * (lane % PR);
    int rkp = 0, rkd = 0;
    auto fetch = [&](int t) {
        const long long row0 = (long long)t * TK;
        if constexpr (SHAPED) {
            if (meta && lane < TK) {
                const int key = (int)row0 + lane;
                rkp = kpos ? kpos[min(key, a.T - 1)] : key;
                rkd = kdoc ? kdoc[min(key, a.T - 1)] : 0;
            }
        }
        if (row0 + TK <= a.T) {
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const char* vp = vb + (row0 + 64 / PR * n) * a.v_row + vlane;
                if constexpr (Q4) {
                    const char* kp = kb + (row0 + 64 / PR * n) * a.k_row + klane;
                    kr[n] = *reinterpret_cast<const u4a2*>(kp + 2);
                    kscale[n] = *reinterpret_cast<const u32a2*>(kp);
                    vr[n] = *reinterpret_cast<const u4a2*>(vp + 2);
                    vscale[n] = *reinterpret_cast<const u32a2*>(vp);
                } else {
                    kr[n] = *reinterpret_cast<const u4a4*>(kb + (row0 + 16 * (n / NB)) * a.k_row + 64 * (n % NB) + klane);
                    vr[n] = *reinterpret_cast<const u4a4*>(vp);
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int vkey = (int)row0 + (lane + 64 * n) / PR, part = (lane + 64 * n) % PR;
                const char* vp = vb + (size_t)min(vkey, a.T - 1) * a.v_row + (Q4 ? 18 : 16) * part;
                if constexpr (Q4) {
                    const char* kp = kb + (size_t)min(vkey, a.T - 1) * a.k_row + 18 * part;
                    kr[n] = *reinterpret_cast<const u4a2*>(kp + 2);
                    kscale[n] = *reinterpret_cast<const u32a2*>(kp);
                    vr[n] = *reinterpret_cast<const u4a2*>(vp + 2);
                    vscale[n] = *reinterpret_cast<const u32a2*>(vp);
                } else {
                    const int kkey = min((int)row0 + 16 * (n / NB) + i, a.T - 1);
                    kr[n] = *reinterpret_cast<const u4a4*>(kb + (size_t)kkey * a.k_row + 64 * (n % NB) + 16 * kg);
                    vr[n] = *reinterpret_cast<const u4a4*>(vp);
                }
            }
        }
    };

    // every splits-th tile is this workgroup's, of those every fourth this wavefront's: what the rows see is spread over all
    const int stride = 4 * a.splits;
    int t = sp + a.splits * wave;
    if (t < t1) fetch(t);  // (before it is known whether a row sees these keys: what it reads is there)

    Row row[NR];
    // (without positions: ascending with the rows)
    int wmin = limitOf(a, a.pos0 + row0 / a.G), wmax = limitOf(a, a.pos0 + (row0 + rows - 1) / a.G);
#pragma unroll
    for (int n = 0; n < NR; ++n) row[n] = rowOf(a, kvh, row0 + 16 * n + i);
    if (SHAPED && a.qpos) {
        wmin = INT_MAX;
        wmax = -1;
#pragma unroll
        for (int n = 0; n < NR; ++n) {  // (rows past the last one repeat it)
            wmin = min(wmin, row[n].limit);
            wmax = max(wmax, row[n].limit);
        }
        wmin = waveMin(wmin);
        wmax = waveMax(wmax);
    }
    if (!kpos) t1 = wmax < 0 ? 0 : min(t1, wmax / TK + 1);

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
        top = swap32Max(swap16Max(top));
        const QScale qs = qScale(top, a.scale);
        c[n] = qs.c;
#pragma unroll
        for (int b = 0; b < NB; ++b) qSplit8(x[b], qs, qh[n][b], ql[n][b]);
    }
    const Shape shape = SHAPED ? shapeOf(a) : Shape{};
    const NibbleMagic magic = nibbleMagic();

    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 o[NR][DT];
    float m[NR], l[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
        for (int d = 0; d < DT; ++d) o[n][d] = zero;
        m[n] = -INFINITY;
        l[n] = 0.0f;
    }
    // the key whose codes this lane addresses in the transposed reads: nibble x of word w of a lane's result is element
    // 2 (x % 4) + x / 4 of tile half w, and element e is key 32 w + 16 (e / 4) + 4 kg + e % 4
    const int xn = i & 7, en = 2 * (xn & 3) + (xn >> 2);
    const int trow = 32 * (i >> 3) + 16 * (en >> 2) + 4 * kg + (en & 3);

    for (; t < t1; t += stride) {
        bool wild = false;
        h8 ka[Q4 ? 1 : 2 * NB];
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int key = (lane + 64 * n) / PR, part = (lane + 64 * n) % PR;
            if constexpr (Q4) {
                *reinterpret_cast<u4*>(mine + key * G::Row + 16 * part) = kr[n];
                *reinterpret_cast<u4*>(mine + G::oV + key * G::Row + 16 * part) = vr[n];
                reinterpret_cast<float*>(mine + G::oS)[part * 64 + key] = finiteOrNaN(halfBits(kscale[n] & 0xFFFFu));
                uint32_t s = t * TK + key < a.T ? vscale[n] & 0xFFFFu : 0u;
                if (wildScale(s)) {
                    s = 0;
                    wild = true;
                }
                // in the order of the products: [block][tile half][kg][16-key half, key % 4]
                const int at = ((part * 2 + (key >> 5)) * 4 + ((key & 15) >> 2)) * 8 + 4 * ((key >> 4) & 1) + (key & 3);
                reinterpret_cast<unsigned short*>(mine + G::oD)[at] = (unsigned short)s;
            } else {
                u4 x = vr[n];
                if (t * TK + key >= a.T) x = u4{0, 0, 0, 0};
                if (wildHalves(x[0]) | wildHalves(x[1]) | wildHalves(x[2]) | wildHalves(x[3])) {
                    wild = true;
#pragma unroll
                    for (int w = 0; w < 4; ++w) x[w] = tameHalves(x[w]);
                }
                *reinterpret_cast<u4*>(mine + key * G::VRow + 16 * part) = x;
                ka[n] = __builtin_bit_cast(h8, kr[n]);
            }
        }
        if constexpr (SHAPED) {
            if (meta && lane < TK) {
                int* mt = reinterpret_cast<int*>(mine + G::oMeta);
                mt[lane] = rkp < 0 || t * TK + lane >= a.T ? kNoKey : rkp;
                mt[TK + lane] = rkd;
            }
        }
        if (t + stride < t1) fetch(t + stride);
        waveLds();
        float x[NR][U * 4];
        if constexpr (Q4) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                f32x4 s[NR][NB];  // all blocks' products before their sums are taken: the matrix unit's latency overlaps
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const h8 kk = nibbles(*reinterpret_cast<const uint32_t*>(mine + (16 * u + i) * G::Row + 16 * b + 4 * kg), magic);
#pragma unroll
                    for (int n = 0; n < NR; ++n) {
                        s[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, qh[n][b], zero, 0, 0, 0);
                        s[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, ql[n][b], s[n][b], 0, 0, 0);
                    }
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const f32x4 d = *reinterpret_cast<const f32x4*>(mine + G::oS + (b * 64 + 16 * u + 4 * kg) * 4);
#pragma unroll
                    for (int n = 0; n < NR; ++n)
#pragma unroll
                        for (int v = 0; v < 4; ++v) x[n][4 * u + v] = b ? fmaf(d[v], s[n][b][v], x[n][4 * u + v]) : d[v] * s[n][b][v];
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
        const bool full = t * TK + TK - 1 <= wmin && t * TK + TK - 1 < a.T;  // (without positions)
        h8 ph[NR][TT], pl[NR][TT];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const float c2 = factor2(c[n]);
            if constexpr (SHAPED) {
                if (shape.inv_cap > 0.0f) {
                    capScores<U * 4>(x[n], capFactor(c[n], shape), shape);
                } else {
#pragma unroll
                    for (int v = 0; v < U * 4; ++v) x[n][v] *= c2;
                }
                const int* mt = reinterpret_cast<const int*>(mine + G::oMeta) + 4 * kg;
                if (shape.bias) {
                    const float slope = -row[n].slope * kLog2e;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int key = t * TK + 16 * u + 4 * kg;
                        int4 p = {key, key + 1, key + 2, key + 3};
                        if (meta) p = *reinterpret_cast<const int4*>(mt + 16 * u);
                        x[n][4 * u] = fmaf(slope, fabsf((float)(row[n].pos - p.x)), x[n][4 * u]);
                        x[n][4 * u + 1] = fmaf(slope, fabsf((float)(row[n].pos - p.y)), x[n][4 * u + 1]);
                        x[n][4 * u + 2] = fmaf(slope, fabsf((float)(row[n].pos - p.z)), x[n][4 * u + 2]);
                        x[n][4 * u + 3] = fmaf(slope, fabsf((float)(row[n].pos - p.w)), x[n][4 * u + 3]);
                    }
                }
                if (a.mask) {
                    const unsigned short* mrow = a.mask + (size_t)row[n].token * a.m_row2;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int key = t * TK + 16 * u + 4 * kg;
                        const uint32_t* mr = reinterpret_cast<const uint32_t*>(mrow) + key / 2;
                        const uint32_t w0 = key < a.T ? mr[0] : 0xFC00FC00u, w1 = key + 2 < a.T ? mr[1] : 0xFC00FC00u;
                        x[n][4 * u] = addMask(x[n][4 * u], w0 & 0xFFFFu);
                        x[n][4 * u + 1] = addMask(x[n][4 * u + 1], w0 >> 16);
                        x[n][4 * u + 2] = addMask(x[n][4 * u + 2], w1 & 0xFFFFu);
                        x[n][4 * u + 3] = addMask(x[n][4 * u + 3], w1 >> 16);
                    }
                }
                if (meta) {  // (keys past the end are at kNoKey)
                    auto unseen = [&](int pos, int doc) { return bool((pos > row[n].limit) | (doc != row[n].doc)); };
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int4 p = *reinterpret_cast<const int4*>(mt + 16 * u), d = *reinterpret_cast<const int4*>(mt + TK + 16 * u);
                        x[n][4 * u] = unseen(p.x, d.x) ? -INFINITY : x[n][4 * u];
                        x[n][4 * u + 1] = unseen(p.y, d.y) ? -INFINITY : x[n][4 * u + 1];
                        x[n][4 * u + 2] = unseen(p.z, d.z) ? -INFINITY : x[n][4 * u + 2];
                        x[n][4 * u + 3] = unseen(p.w, d.w) ? -INFINITY : x[n][4 * u + 3];
                    }
                }
            }
            if (!meta && !full) {
                const int last = min(row[n].limit, a.T - 1) - t * TK - 4 * kg;
#pragma unroll
                for (int v = 0; v < U * 4; ++v) x[n][v] = 16 * (v >> 2) + (v & 3) <= last ? x[n][v] : -INFINITY;
            }
            float bm = x[n][0];
#pragma unroll
            for (int v = 1; v < U * 4; ++v) bm = fmaxf(bm, x[n][v]);
            bm = swap32Max(swap16Max(bm));
            if constexpr (!SHAPED) bm *= c2;
            const bool ahead = bm > m[n] + kLag;
            if (__any(ahead)) {
                const float mn = ahead ? bm : m[n], alpha = ahead ? ex2(m[n] - mn) : 1.0f;
                l[n] *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[n][d] *= alpha;
                m[n] = mn;
            }
            const float off = kPBits - (m[n] == -INFINITY ? 0.0f : m[n]);
            float ls = 0.0f;
#pragma unroll
            for (int v = 0; v < U * 4; ++v) {
                x[n][v] = ex2(SHAPED ? x[n][v] + off : fmaf(x[n][v], c2, off));
                ls += x[n][v];
            }
            l[n] += ls;
            splitParts<U * 4>(x[n], ph[n], pl[n]);
        }
        if (__builtin_expect(__any(wild), 0)) {  // values that are no matrix operands, for the rows that see them
            float* zr = reinterpret_cast<float*>(mine + G::oZ);
#pragma unroll 1
            for (int key = 0; key < TK; ++key) {
                const char* vrow = vb + (size_t)min(t * TK + key, a.T - 1) * a.v_row;
                const int xi = 4 * (key >> 4) + (key & 3), from = i + 16 * ((key >> 2) & 3);
#pragma unroll
                for (int e = 0; e < D / 64; ++e) zr[lane + 64 * e] = wildValue<Q4>(vrow, lane + 64 * e);
                waveLds();
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    const float p = __shfl(pick<U * 4>(x[n], xi), from);
                    if (!__any(p != 0.0f)) continue;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            const int rr = 4 * kg + v;
                            const float y = fmaf(p, zr[Q4 ? 32 * (d >> 1) + 8 * (d & 1) + (rr >> 1) + 16 * (rr & 1) : 16 * d + rr], o[n][d][v]);
                            o[n][d][v] = p != 0.0f ? y : o[n][d][v];
                        }
                }
                waveLds();
            }
        }
        if constexpr (Q4) {
            const unsigned short* vd = reinterpret_cast<const unsigned short*>(mine + G::oD);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                h8 dd[2];
#pragma unroll
                for (int w = 0; w < 2; ++w) dd[w] = *reinterpret_cast<const h8*>(vd + ((b * 2 + w) * 4 + kg) * 8);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int d = 2 * b + s;
                    const i2 w2 = __builtin_amdgcn_ds_read_tr4_b64_v2i32((LdsI2)(mine + G::oV + trow * G::Row + 8 * d));
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const h8 code = nibbles((uint32_t)w2[w], magic);
                        const h8 vh = code * dd[w], vl = __builtin_elementwise_fma(code, dd[w], -vh);
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
    bool lost = false;
    for (int x = tid; x < rows * (D / 4); x += 256) {  // four values each
        const int r = x / (D / 4), at = x % (D / 4) * 4;
        float mw[4], lw[4], M = -INFINITY, L = 0.0f;
        f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f}, ow[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float2 ml = *reinterpret_cast<const float2*>(jm + 2 * (w * NR * 16 + r));
            mw[w] = ml.x;
            lw[w] = ml.y;
            ow[w] = *reinterpret_cast<const f32x4*>(jo + (w * NR * 16 + r) * G::ORow + at);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, mw[w]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = mw[w] == -INFINITY ? 0.0f : ex2(mw[w] - M);
            L = fmaf(f, lw[w], L);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = f != 0.0f ? fmaf(f, ow[w][e], y[e]) : y[e];
        }
        lost |= L != L;
        float* dst;
        if (a.splits == 1) {
            const int token = (row0 + r) / a.G, head = kvh * a.G + (row0 + r - token * a.G);
            dst = a.out + ((size_t)token * a.H + head) * D;
            y *= L == 0.0f ? 0.0f : 1.0f / L;
            if (a.lse && at == 0) a.lse[(size_t)token * a.H + head] = L == 0.0f ? -INFINITY : fmaf(M, kLn2, logf(L * kPInv));
        } else {
            const size_t pr = ((size_t)sp * a.H_kv + kvh) * a.rows + row0 + r;
            dst = a.part + pr * D;
            y *= kPInv;
            if (at == 0) {
                float* ml = a.part + (size_t)a.splits * a.H_kv * a.rows * D + 2 * pr;
                ml[0] = M;
                ml[1] = L * kPInv;
            }
        }
        if constexpr (Q4) {  // values 8 (rr / 16) + rr / 2 + 16 (rr % 2) of the block, rr = at .. at + 3 in the block
            float* to = dst + (at & ~31) + 8 * ((at >> 4) & 1) + ((at & 15) >> 1);
            *reinterpret_cast<f2a4*>(to) = f32x2{y[0], y[2]};
            *reinterpret_cast<f2a4*>(to + 16) = f32x2{y[1], y[3]};
        } else {
            *reinterpret_cast<f4a4*>(dst + at) = y;
        }
    }
    if (__builtin_expect(__any(lost), 0)) {  // of the rows that this wavefront has written
        __threadfence();
        for (int r = 0; r < rows; ++r) {
            float L = 0.0f;
            for (int w = 0; w < 4; ++w) L += jm[2 * ((w * NR) * 16 + r) + 1];
            if (r * (D / 4) / 64 % 4 == wave && L != L) writePlainRow<D, Q4, TK>(kvh, row0 + r, sp, lane);
        }
    }
}

// ---------------------------------------------------------------------------------------------- joining key ranges
// o = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) for each row. A thread takes four of a row's values in every SG-th range,
// the first of its loads issued before the weights are known; the row's threads share the weights, and the SG sums are
// added in order through LDS. What counts is the latency of a round trip: 2.9 to 4.2 us for 32 rows of 32 or 64 ranges.
template <int D, int SG>
__global__ __launch_bounds__(256) void flash_ext_join_kernel(FxParams a) {
    constexpr int LP = D / 4, RT = LP * SG, RPB = 256 / RT;  // lanes to a row's values, threads to a row, rows to a workgroup
    constexpr int Ahead = 8, Most = 512;                     // (fxPlan: no more ranges)
    __shared__ f32x4 sum[SG > 1 ? 256 : 1];
    __shared__ float wt[SG > 1 ? RPB : 1][SG > 1 ? Most : 1], red[2][4];
    const int tid = threadIdx.x, q = tid % RT, at = q % LP, g = q / LP, x = tid / RT;
    const int total = a.H_kv * a.rows, n = blockIdx.x * RPB + x, nr = min(n, total - 1);  // row n % rows of KV head n / rows
    const float* po = a.part + (size_t)nr * D + 4 * at;
    const float* ml = a.part + (size_t)a.splits * total * D + 2 * (size_t)nr;
    f32x4 z[Ahead];
#pragma unroll
    for (int k = 0; k < Ahead; ++k) z[k] = *reinterpret_cast<const f4a4*>(po + (size_t)min(g + SG * k, a.splits - 1) * total * D);
    float M = -INFINITY, L = 0.0f;
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (SG == 1) {
        float ms[4], ls[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            ms[s] = s < a.splits ? ml[(size_t)s * total * 2] : -INFINITY;
            ls[s] = s < a.splits ? ml[(size_t)s * total * 2 + 1] : 0.0f;
            M = fmaxf(M, ms[s]);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const float f = ms[s] == -INFINITY ? 0.0f : ex2(ms[s] - M);
            L = fmaf(f, ls[s], L);
            if (f != 0.0f) y += f * z[s];
        }
    } else {
        for (int s = q; s < a.splits; s += RT) {
            const float ms = ml[(size_t)s * total * 2];
            wt[x][s] = ms;
            M = fmaxf(M, ms);
        }
        M = waveMaxF(M);
        if ((tid & 63) == 0) red[0][tid >> 6] = M;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < RT / 64; ++w) M = fmaxf(M, red[0][x * (RT / 64) + w]);
        for (int s = q; s < a.splits; s += RT) {
            const float ms = wt[x][s], f = ms == -INFINITY ? 0.0f : ex2(ms - M);
            L = fmaf(f, ml[(size_t)s * total * 2 + 1], L);
            wt[x][s] = f;
        }
        L = waveSumF(L);
        if ((tid & 63) == 0) red[1][tid >> 6] = L;
        __syncthreads();
        L = 0.0f;
#pragma unroll
        for (int w = 0; w < RT / 64; ++w) L += red[1][x * (RT / 64) + w];
#pragma unroll
        for (int k = 0; k < Ahead; ++k) {
            const int s = g + SG * k;
            const float f = s < a.splits ? wt[x][s] : 0.0f;
            if (f != 0.0f) y += f * z[k];
        }
        for (int s = g + SG * Ahead; s < a.splits; s += SG) {
            const float f = wt[x][s];
            const f32x4 w = *reinterpret_cast<const f4a4*>(po + (size_t)s * total * D);
            if (f != 0.0f) y += f * w;
        }
        sum[tid] = y;
        __syncthreads();
        if (g) return;
#pragma unroll
        for (int k = 1; k < SG; ++k) y += sum[tid + k * LP];
    }
    if (n >= total) return;
    const int kvh = n / a.rows, r = n - kvh * a.rows, token = r / a.G, head = kvh * a.G + (r - token * a.G);
    const float f = L == 0.0f ? 0.0f : 1.0f / L;
    *reinterpret_cast<f4a4*>(a.out + ((size_t)token * a.H + head) * D + 4 * at) = y * f;
    if (a.lse && at == 0) a.lse[(size_t)token * a.H + head] = L == 0.0f ? -INFINITY : fmaf(M, kLn2, logf(L));
}

template <class F>
int allow(F* kernel, int lds) {
    return fromHip(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds),
                   "flash_ext: LDS size");
}

template <int D, int SG>
int join(const FxParams& p, hipStream_t s) {
    constexpr int rows = 256 / (D / 4) / SG;
    hipLaunchKernelGGL((flash_ext_join_kernel<D, SG>), dim3((p.H_kv * p.rows + rows - 1) / rows), dim3(256), 0, s, p);
    return fromHip(hipGetLastError(), "flash_ext (join)");
}

template <int D, bool Q4, bool SHAPED>
int run(const FxParams& p, const FxPlan& plan, hipStream_t s) {
    if (plan.few) {
        constexpr int NR2 = D == 256 ? 1 : 2;  // (16 rows of 256 values fill the registers)
        const dim3 grid(p.splits, p.H_kv, (p.rows + 16 * NR2 - 1) / (16 * NR2));
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
        using G = Geo<D, Q4>;
        static const int ok = allow(flash_ext_kernel<D, Q4, SHAPED>, G::Lds);
        if (ok) return ok;
        hipLaunchKernelGGL((flash_ext_kernel<D, Q4, SHAPED>), dim3(p.H_kv, (p.rows + 127) / 128, p.splits), dim3(G::Threads), G::Lds, s, p);
    }
    if (int e = fromHip(hipGetLastError(), "flash_ext")) return e;
    // two to four ranges: a thread adds them up; more: the row's threads share them
    if (p.splits > 4) return join<D, D == 256 ? 4 : 8>(p, s);
    return p.splits > 1 ? join<D, 1>(p, s) : 0;
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
    // (positions of queries too: the unshaped kernels take what their rows see from pos0)
    const bool shaped = a.mask || a.qpos || a.kpos || a.kdoc || a.slopes || a.softcap > 0.0f;
    switch (a.d.D) {
        case 64: return runD<64>(q4, shaped, p, plan, s);
        case 128: return runD<128>(q4, shaped, p, plan, s);
        case 256: return runD<256>(q4, shaped, p, plan, s);
        default: return fromHip(hipErrorInvalidValue, "flash_ext: D");
    }
}

}  // namespace kcamd
