// kflash_pages.hip -- flash_pages_f16 (gfx950): attention of a step's tokens (single tokens, chunks of prompts, drafted trees) of many
// sequences over an fp16 paged cache,
//   x_ij = log2 e scale q_i.k_j,   o_i = sum_j 2^(x_ij - m_i) v_j / l_i,   m_i = max_j x_ij, l_i = sum_j 2^(x_ij - m_i)
// over the positions j that token i sees, in one pass over the keys with running m and l.
//
// The lengths are known on the device alone. So the host launches as many workgroups as run at once, and these share out the work by
// themselves: the rows (token, query head of the group) of a sequence and KV head in blocks of RT, "items", each of the steps that its
// sequence's length gives; all items' steps in a row are divided evenly among the workgroups. An item whose steps fall to several
// workgroups is joined by a second kernel from their sums (in the order of the keys, so that results do not depend on
// which workgroup was first).
//
// What bounds it: single tokens the cache's bytes (128 sequences of 4000 positions, 32 heads on 8 of 128: 363 us with the join, 5.7 TB/s); wide trees products
// of split operands and softmax, which a SIMD's two wavefronts hardly overlap (64 nodes over 100000 positions: 220 us, 0.48 PFLOP/s
// counted once; in calls back to back 237; matrix units busy in 47% of the cycles, vector instructions in 43%); a small call the chain of
// shares, first loads, steps and join (one token over 8191 positions: 12 + 4 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "internal.hpp"
#include "kflash_ext_device.hpp"
#include "kserve.hpp"

namespace kcamd {
namespace {

using namespace fx;

// (as in kflash_ext.hip: a row's m may lag behind its maximum by kLag; p is split into fp16 parts at the scale 2^kPBits)
constexpr float kLag = 4.0f, kPBits = 11.0f, kPInv = 1.0f / 2048.0f;

struct FpParams {
    const float* q;
    const char *k, *v;
    const int *table, *start, *len, *tree;
    float *out, *lse;
    int* head;    // workspace: the number of items, then each item's description (8 ints)
    float* part;  // and two sums for each workgroup: of the item it begins in the middle of, and of the one it does not end
    long long k_row, k_head, v_row, v_head;
    int H, H_kv, G, N, seqs, shift, max_pages, n_pages, tree_words, q_tok, q_head, table_row, groups, items;
    float scale;
};

struct Item {
    int token0, nodes, len, base;  // the sequence's first token, its tokens, its positions, those before the tokens
    int r0, rows, kvh;             // the item's first row, the sequence's rows
    const int* table;
};

// Which 32 of a row's bits from bit `at` on are set in its words (at may be negative: bits below 0 are set).
__device__ __forceinline__ uint32_t windowOf(uint32_t w0, uint32_t w1, const int* words, int n, int at) {
    auto word = [&](int i) -> uint32_t { return i < 0 ? ~0u : i == 0 ? w0 : i == 1 ? w1 : i < n ? (uint32_t)words[i] : 0u; };
    const int i = at >> 5, s = at & 31;
    if (i < -1) return ~0u;
    const unsigned long long both = (unsigned long long)word(i + 1) << 32 | word(i);
    return (uint32_t)(both >> s);
}

// The slot of a position, -1 where it has none.
__device__ __forceinline__ long long slotOf(const FpParams& a, const Item& it, int pos) {
    const int page = it.table[pos >> a.shift];
    return page < 0 || page >= a.n_pages ? -1ll : ((long long)page << a.shift) + (pos & ((1 << a.shift) - 1));
}

// Row r of an item over positions [p0, p1) by a wavefront, from the definition in plain f32: values lane + 64 e of the sum of
// 2^(x - m) v to o. For rows whose sums on the matrix cores met an infinity or NaN.
template <int D>
__device__ __forceinline__ void plainRow(const FpParams& a, const Item& it, int r, int p0, int p1, int lane, float& m, float& l, float (&o)[D / 64]) {
    const int node = r / a.G, token = it.token0 + node, head = it.kvh * a.G + (r - node * a.G);
    const float* q = a.q + (long long)token * a.q_tok + (long long)head * a.q_head;
    const int* words = a.tree ? a.tree + (size_t)token * a.tree_words : nullptr;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] = 0.0f;
    for (int k0 = p0; k0 < p1; k0 += 64) {
        const int pos = k0 + lane, j = pos - it.base;
        bool seen = pos < p1 && pos < it.len;
        if (seen && j >= 0) seen = words ? j < 32 * a.tree_words && ((uint32_t)words[j >> 5] >> (j & 31) & 1u) : j <= node;
        const long long slot = seen ? slotOf(a, it, pos) : -1;
        float x = -INFINITY;
        if (slot >= 0) {
            const char* k = a.k + slot * a.k_row + it.kvh * a.k_head;
            x = 0.0f;
#pragma unroll 4
            for (int d = 0; d < D; ++d) x = fmaf(q[d] * a.scale, halfBits(loadHalf(k + 2 * d)), x);
            x *= kLog2e;
        }
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
            const long long s = (long long)(((unsigned long long)(unsigned)__shfl((int)(slot >> 32), at) << 32) | (unsigned)__shfl((int)slot, at));
            const char* v = a.v + s * a.v_row + it.kvh * a.v_head;
#pragma unroll
            for (int e = 0; e < D / 64; ++e) o[e] = fmaf(pk, halfBits(loadHalf(v + 2 * (lane + 64 * e))), o[e]);
        }
    }
}

// A form of the kernel: W wavefronts of 16 NR rows, at most KM of them side by side over the keys.
typedef __attribute__((address_space(3))) void* LdsPtr;
// V^T of 64 of the head's values (4 operands) from value 64 J on, and its products. The transposed reads are written out: before
// each of the builtin's the compiler waits for all loads into LDS under way.
template <int D, int NR, int J>
__device__ __forceinline__ void valuesTimesP(const uint32_t (&at)[4], const h8 (&ph)[NR], const h8 (&pl)[NR], f32x4 (&o)[NR][D / 16]) {
    s4 x[4], y[4];
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %4, %8 offset:%13\n\t"
        "ds_read_b64_tr_b16 %1, %9 offset:%12\n\tds_read_b64_tr_b16 %5, %9 offset:%13\n\t"
        "ds_read_b64_tr_b16 %2, %10 offset:%12\n\tds_read_b64_tr_b16 %6, %10 offset:%13\n\t"
        "ds_read_b64_tr_b16 %3, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(y[0]), "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(128 * J), "n"(128 * J + 16 * 2 * D)
        : "memory");
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const h8 va = __builtin_bit_cast(h8, __builtin_shufflevector(x[d], y[d], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            o[n][4 * J + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[n], o[n][4 * J + d], 0, 0, 0);
            o[n][4 * J + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[n], o[n][4 * J + d], 0, 0, 0);
        }
    }
    if constexpr (64 * (J + 1) < D) valuesTimesP<D, NR, J + 1>(at, ph, pl, o);
}

template <int D, int NR, int W, int KM>
struct FpGeo {
    static constexpr int RT = 16 * NR * W, Threads = 64 * W;  // rows of an item, at most
    static constexpr int Tile = 2 * 32 * 2 * D;               // bytes of 32 keys and values
    static constexpr int ORow = D + 4;                        // the join of the wavefronts: floats of a row
    static constexpr int Loop = 2 * KM * Tile, Join = KM > 1 ? RT * (ORow + 2) * 4 : 0;
    static constexpr int Lds = Loop > Join ? Loop : Join;
    static constexpr int Part = RT * (D + 2);                 // floats of a sum: rows of D values, then m and l of each
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t bufRes(const char* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), (short)0, bytes, 0x00020000);
}
// A key's or value's row lies in LDS with its 16-byte chunks permuted: chunk c at c ^ rowBits(row), so that eight consecutive rows' reads
// of one chunk, and four rows' transposed reads of two, are on different banks.
__device__ __forceinline__ constexpr int rowBits(int row) { return (row & 3) << 1 | (row >> 2 & 1); }

// A sequence of few rows has them in few wavefronts, and the others take other keys: RG wavefronts (a power of two) with 16 NR rows each,
// KG = W / RG of these groups with 32 keys of a step each, RG the least that holds the rows (and leaves KG at most KM, for
// which there is LDS).
// Matrix form (v_mfma_f32_16x16x32_f16; lane (i, g), i < 16, g < 4):
//   S^T = K Q^T: A = 16 keys (LDS; lane: key i, values 32 b + 8 g ..), B = q hi / lo (registers; row i). Lane holds keys 4 g + v of row i.
//   O^T += V^T P^T: A = V^T by transposed LDS reads, B = p hi / lo, the score registers as they are: the products' index 8 g + e
//   stands for key 16 (e / 4) + 4 g + e % 4.
// Keys and values come by buffer-to-LDS loads, a step ahead, with a resource for each 16 positions (a page holds 16 at least) that
// ends with the last valid one: what lies behind it in the page reads as zeros.
template <int D, int NR, int W, int KM>
__global__ __launch_bounds__(64 * W, W > KM ? 2 : 1) void flash_pages_kernel(FpParams a) {
    using G = FpGeo<D, NR, W, KM>;
    constexpr int NB = D / 32, DT = D / 16, RT = G::RT, NT = G::Threads;
    extern __shared__ int4 lds4[];
    char* lds = reinterpret_cast<char*>(lds4);
    __shared__ long long found[4];
    __shared__ long long scan[2][W];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int wg = blockIdx.x;

    // ---- this workgroup's share. Four units are what 32 positions of a KV head cost where the wavefronts stand side by side over the keys as
    // much as they can (the cache's bytes bound that); positions of more rows cost more, and an item's first loads, its q and its join as much as
    // Setup units, where it is not many workgroups that take an item. (us with one price for all positions, with these, with the items' own too,
    // 32 heads on 8 of 128: trees of 8 to 24 nodes, 32 sequences of 4000 positions 150, 137, 134, 128 of 2000 307, 280, 275; trees of 20 to
    // 64 nodes, where twice the price for more than 128 rows was too much, 279, 256, 249 and 533, 496, 473; one to seven tokens 129, 115,
    // 113; single tokens of 128 sequences 196 and 189.)
    constexpr int lgW = W == 8 ? 3 : 2, lgMin = W / KM == 4 ? 2 : W / KM == 2 ? 1 : 0, lgRows = NR == 2 ? 5 : 4;
    constexpr int Setup = 24;
    auto tileUnits = [](int lg) { return W == 8 ? (lg < lgW ? 4 : D == 256 ? 6 : 7) : 4 + 2 * (lg - lgMin); };
    static_assert(1 << lgW == W && KM << lgMin == W && 1 << lgRows == 16 * NR);
    // A block of rows counts with all of its sequence's steps, also where its last row sees fewer (a prompt's chunk: 2048 tokens on none 158 us, 220
    // TFLOP/s of the seen pairs, on 2048 278 and 370; 512 on none 31).
    struct Seq {
        int nodes, len, lg, blocks, steps, weight;  // tokens, positions, log2 RG, blocks of rows, steps, a step's units
        long long units;                            // of all its items' steps
    };
    const int most = a.max_pages << a.shift;
    auto sequence = [&](int s) {
        Seq q;
        const int x = min(max(a.start[s], 0), a.N), y = min(max(a.start[s + 1], 0), a.N);
        q.nodes = max(0, y - x);
        q.len = min(max(a.len[s], 0), most);
        const int waves = (q.nodes * a.G + (1 << lgRows) - 1) >> lgRows;
        q.lg = min(max(waves > 1 ? 32 - __builtin_clz(waves - 1) : 0, lgMin), lgW);
        q.blocks = (waves + (1 << q.lg) - 1) >> q.lg;
        const int sh = 5 + lgW - q.lg;
        q.steps = max(1, (q.len >> sh) + ((q.len & ((1 << sh) - 1)) != 0));
        q.weight = (W >> q.lg) * tileUnits(q.lg);
        q.units = (long long)q.blocks * a.H_kv * ((long long)q.steps * q.weight);
        return q;
    };
    // (sums up to and with this thread's of its sequences' units and items, and over all threads)
    long long total = 0, items = 0, mine = 0, upTo = 0, itemsTo = 0;
    int myItems = 0;
    auto round = [&](int s0) {
        mine = myItems = 0;
        if (s0 + tid < a.seqs) {
            const Seq q = sequence(s0 + tid);
            mine = q.units;
            myItems = q.blocks * a.H_kv;
        }
        long long x = mine, y = myItems;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const long long z = __shfl_up(x, o), w = __shfl_up(y, o);
            if (lane >= o) {
                x += z;
                y += w;
            }
        }
        __syncthreads();
        if (lane == 63) {
            scan[0][wave] = x;
            scan[1][wave] = y;
        }
        __syncthreads();
        upTo = total + x;
        itemsTo = items + y;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            upTo += w < wave ? scan[0][w] : 0;
            itemsTo += w < wave ? scan[1][w] : 0;
            total += scan[0][w];
            items += scan[1][w];
        }
    };
    for (int s0 = 0; s0 < a.seqs; s0 += NT) round(s0);
    if (wg == 0 && tid == 0) a.head[0] = (int)min(items, (long long)a.items);
    const int setup = items * 8 >= a.groups ? Setup : 0;
    total += items * setup;
    // (a workgroup's units hold a step at least of each item whose steps they touch: as many as a step has at most, and a power of two of
    // workgroups)
    // (few items: whole steps of most kinds, so that an item's last workgroup rather ends with it than begins the next)
    long long share = max(4ll * W, (total + a.groups - 1) >> (31 - __builtin_clz(a.groups)));
    if (!setup) share = (share + 7) & ~7ll;
    const long long u0 = wg * share, u1 = min(total, u0 + share);
    if (u0 >= u1) return;
    // the sequence of unit u0, the units and items before it
    auto find = [&](int s0) {
        const long long to = upTo + itemsTo * setup, from = to - mine - myItems * setup;
        if (u0 >= from && u0 < to) {
            found[0] = s0 + tid;
            found[1] = from;
            found[2] = itemsTo - myItems;
        }
    };
    if (a.seqs <= NT) {
        find(0);
    } else {
        total = items = 0;
        for (int s0 = 0; s0 < a.seqs; s0 += NT) {
            round(s0);
            find(s0);
        }
    }
    __syncthreads();
    int s = __builtin_amdgcn_readfirstlane((int)found[0]);
    long long sBefore = found[1];
    int sItems = __builtin_amdgcn_readfirstlane((int)min(found[2], (long long)a.items));
    // x / y, x mostly small
    auto over = [](long long x, long long y) { return x >> 31 || y >> 31 ? (int)(x / y) : (int)((unsigned)x / (unsigned)y); };

    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    // a lane's share of a load's addresses (64 chunks of 16 bytes: RPL rows)
    constexpr int CPR = D / 8, RPL = 64 / CPR, LPT = 32 / RPL;
    const int chunk = 16 * (lane % CPR ^ rowBits(lane / CPR)), klane = lane / CPR * (int)a.k_row, vlane = lane / CPR * (int)a.v_row;

    for (long long u = u0; u < u1;) {
        // ---- the item of unit u
        Seq q = sequence(s);
        const auto all = [&] { return q.units + (long long)q.blocks * a.H_kv * setup; };
        while (u >= sBefore + all()) {
            sBefore += all();
            sItems += q.blocks * a.H_kv;
            q = sequence(++s);
        }
        const int RG = 1 << q.lg, KG = W >> q.lg, Step = 32 * KG, rg = wave & (RG - 1), kg = wave >> q.lg;
        const int rt = (16 * NR) << q.lg;
        char* tiles = lds + kg * 2 * G::Tile;
        Item it;
        it.token0 = min(max(a.start[s], 0), a.N);
        it.nodes = q.nodes;
        it.len = q.len;
        it.base = a.len[s] - q.nodes;
        it.rows = q.nodes * a.G;
        it.table = a.table + (size_t)s * a.table_row;
        const long long per = (long long)q.steps * q.weight + setup;  // an item's units
        const int at = over(u - sBefore, per);
        const long long i0 = sBefore + at * per;
        const int item = sItems + at;
        it.kvh = at / q.blocks;
        it.r0 = (at - it.kvh * q.blocks) * rt;
        // the steps whose first unit is in this workgroup's share
        auto stepsBefore = [&](long long x) { return (int)((unsigned)(max(x - setup, 0ll) + q.weight - 1) / (unsigned)q.weight); };
        const int st0 = stepsBefore(u - i0), st1 = stepsBefore(min(u1 - i0, per));
        const bool whole = st0 == 0 && st1 == q.steps;
        const int rows = min(rt, it.rows - it.r0);
        u = min(u1, i0 + per);
        if (item >= a.items) return;  // (more rows than N tokens have: sequences that overlap)
        if (st0 >= st1) continue;     // (the item's last steps began in the share before, or its first ones begin in the next)
        if (st0 == 0 && tid < 8) {
            const int n = over(i0 + setup + (long long)(q.steps - 1) * q.weight - u0, share) + 1;
            const int d[8] = {it.token0, it.r0, rows, it.kvh, wg, n, 0, 0};
            a.head[4 + 8 * item + tid] = d[tid];
        }
        // steps that some row sees
        const int lastNode = (it.r0 + rows - 1) / a.G;
        const int vis = a.tree ? it.len : (int)min((long long)it.len, max(0ll, (long long)it.base + lastNode + 1));
        const int end = min(st1, vis / Step + (vis % Step != 0));

        // ---- loads
        const char* kb = a.k + it.kvh * a.k_head;
        const char* vb = a.v + it.kvh * a.v_head;
        int window = 0, win0 = -1000;  // entries win0 + lane of the table row
        // (returns which of the 32 positions there are)
        auto issue = [&](int st, int slot) -> uint32_t {
            const int p0 = st * Step, first = p0 >> a.shift;
            if (first < win0 || ((p0 + Step - 1) >> a.shift) >= win0 + 64) {
                win0 = first;
                window = it.table[min(win0 + lane, a.max_pages - 1)];
            }
            const int key0 = p0 + 32 * kg;
            if (key0 >= vis) return 0;
            uint32_t valid = 0;
            // 16 positions' first slot (0 without a page), and how many of them there are
            auto half = [&](int h, int& slot0) {
                const int key = key0 + 16 * h;
                const int page = __builtin_amdgcn_readlane(window, (key >> a.shift) - win0 & 63);
                const bool in = key < it.len && page >= 0 && page < a.n_pages;
                const int n = in ? min(16, it.len - key) : 0;
                valid |= ((1u << n) - 1) << 16 * h;
                slot0 = in ? (page << a.shift) + (key & ((1 << a.shift) - 1)) : 0;
                return n;
            };
            int s0, s1;
            const int n0 = half(0, s0), n1 = half(1, s1);
            char* to = tiles + slot * G::Tile;
            for (int L = rg; L < LPT; L += RG) {
                const bool second = L >= LPT / 2;
                const int n = second ? n1 : n0, bits = 16 * rowBits(L * RPL & 7), row = L * RPL & 15;
                const long long at = second ? s1 : s0;
                // (the sizes in scalar registers: without it a load is a loop over the lanes' resources)
                const auto rk = bufRes(kb + at * (int)a.k_row, __builtin_amdgcn_readfirstlane(n ? (n - 1) * (int)a.k_row + 2 * D : 0));
                const auto rv = bufRes(vb + at * (int)a.v_row, __builtin_amdgcn_readfirstlane(n ? (n - 1) * (int)a.v_row + 2 * D : 0));
                char *kl = to + L * 1024, *vl = kl + G::Tile / 2;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (LdsPtr)kl, 16, (chunk ^ bits) + klane + row * (int)a.k_row, 0, 0, 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (LdsPtr)vl, 16, (chunk ^ bits) + vlane + row * (int)a.v_row, 0, 0, 0);
            }
            return valid;
        };
        uint32_t valid = 0, validNext = 0;
        if (st0 < end) validNext = issue(st0, 0);

        // ---- the rows
        int node[NR];
        const int* words[NR];
        uint32_t w0[NR], w1[NR];
        h8 qh[NR][NB], ql[NR][NB];
        float c2[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int r = it.r0 + min((rg * NR + n) * 16 + i, rows - 1);
            node[n] = r / a.G;
            const int token = it.token0 + node[n], head = it.kvh * a.G + (r - node[n] * a.G);
            words[n] = a.tree ? a.tree + (size_t)token * a.tree_words : nullptr;
            w0[n] = a.tree ? words[n][0] : 0;
            w1[n] = a.tree && a.tree_words > 1 ? words[n][1] : 0;
            const float* qp = a.q + (long long)token * a.q_tok + (long long)head * a.q_head + 8 * g;
            float x[NB][8], top = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const f32x4 y = *reinterpret_cast<const f4a4*>(qp + 32 * b), z = *reinterpret_cast<const f4a4*>(qp + 32 * b + 4);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[b][e] = e < 4 ? y[e & 3] : z[e & 3];
                    top = fmaxf(top, fabsf(x[b][e]));
                }
            }
            top = swap32Max(swap16Max(top));
            const QScale qs = qScale(top, a.scale);
            c2[n] = factor2(qs.c);
#pragma unroll
            for (int b = 0; b < NB; ++b) qSplit8(x[b], qs, qh[n][b], ql[n][b]);
        }
        f32x4 o[NR][DT];
        float m[NR], l[NR];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
#pragma unroll
            for (int d = 0; d < DT; ++d) o[n][d] = zero;
            m[n] = -INFINITY;
            l[n] = 0.0f;
        }

        // ---- the steps
        const bool idle = rg * NR * 16 >= rows;  // (it loads for the others)
        int slot = 0;
        for (int st = st0; st < end; ++st, slot ^= 1) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (KM < W || RG > 1) __syncthreads();  // every wavefront's loads are there, and the other buffer has been read
            valid = validNext;
            if (st + 1 < end) validNext = issue(st + 1, slot ^ 1);
            const int key0 = st * Step + 32 * kg;
            if (key0 >= vis || idle) continue;
            const char* kt = tiles + slot * G::Tile;
            const char* vt = kt + G::Tile / 2;
            float x[NR][8];
            // (2 NR independent sums, and a wavefront in its products before one in its weights: 240 to 230 us for 64 nodes over 100000
            // positions, 155 to 148 for trees of 32 sequences; two sums took the products' latency each time)
            f32x4 sc[2][NR];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int n = 0; n < NR; ++n) sc[t][n] = zero;
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                h8 ka[2];
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    ka[t] = *reinterpret_cast<const h8*>(kt + (16 * t + i) * 2 * D + 16 * ((4 * b + g) ^ rowBits(i)));
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int n = 0; n < NR; ++n) sc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[t], ql[n][b], sc[t][n], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int n = 0; n < NR; ++n) sc[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[t], qh[n][b], sc[t][n], 0, 0, 0);
            }
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int v = 0; v < 4; ++v) x[n][4 * t + v] = sc[t][n][v];
            // what is not seen
            if (valid != ~0u || key0 + 32 > it.base) {
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    uint32_t seen;
                    if (a.tree) {
                        seen = windowOf(w0[n], w1[n], words[n], a.tree_words, key0 - it.base);
                    } else {
                        const int k = it.base + node[n] + 1 - key0;
                        seen = k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1;
                    }
                    seen = (seen & valid) >> 4 * g;
#pragma unroll
                    for (int v = 0; v < 8; ++v) x[n][v] = seen >> (16 * (v >> 2) + (v & 3)) & 1u ? x[n][v] : -INFINITY;
                }
            }
            h8 ph[NR], pl[NR];
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                // (a lane's own keys first: the row's maximum over its four lanes is only needed where one of them runs ahead)
                float bm = x[n][0];
#pragma unroll
                for (int v = 1; v < 8; ++v) bm = fmaxf(bm, x[n][v]);
                bm *= c2[n];
                if (__any(bm > m[n] + kLag)) {
                    bm = swap32Max(swap16Max(bm));
                    const bool ahead = bm > m[n] + kLag;
                    const float mn = ahead ? bm : m[n], alpha = ahead ? ex2(m[n] - mn) : 1.0f;
                    l[n] *= alpha;
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[n][d] *= alpha;
                    m[n] = mn;
                }
                const float off = kPBits - (m[n] == -INFINITY ? 0.0f : m[n]);
                float ls = 0.0f;
#pragma unroll
                for (int v = 0; v < 8; ++v) {
                    x[n][v] = ex2(fmaf(x[n][v], c2[n], off));
                    ls += x[n][v];
                }
                l[n] += ls;
                h8 hi[1], lo[1];
                splitParts<8>(x[n], hi, lo);
                ph[n] = hi[0];
                pl[n] = lo[0];
            }
            const int vr = 4 * g + (i >> 2);  // (rows vr and vr + 16 have the same bits)
            uint32_t at[4];
#pragma unroll
            for (int d = 0; d < 4; ++d)
                at[d] = (uint32_t)(uintptr_t)(LdsPtr)(vt + vr * 2 * D + 16 * ((2 * d + (i >> 1 & 1)) ^ rowBits(vr)) + 8 * (i & 1));
            valuesTimesP<D, NR, 0>(at, ph, pl, o);
        }

        // ---- the item's rows: to out, or to this workgroup's sums
        float* part = a.part + (2ll * wg + (st0 == 0)) * G::Part;
        auto rowOut = [&](int r, float*& dst) {  // (r: in the item)
            const int rr = it.r0 + r, nd = rr / a.G;
            dst = whole ? a.out + ((size_t)(it.token0 + nd) * a.H + it.kvh * a.G + (rr - nd * a.G)) * D : part + r * D;
        };
        auto rowSums = [&](int r, float M, float L) {
            const int rr = it.r0 + r, nd = rr / a.G;
            if (!whole) {
                part[RT * D + 2 * r] = M;
                part[RT * D + 2 * r + 1] = L;
            } else if (a.lse) {
                a.lse[(size_t)(it.token0 + nd) * a.H + it.kvh * a.G + (rr - nd * a.G)] = L == 0.0f ? -INFINITY : fmaf(M, kLn2, logf(L));
            }
        };
        auto again = [&](int r) {  // a row that met an infinity or NaN
            float M, L, y[D / 64], *dst;
            plainRow<D>(a, it, it.r0 + r, st0 * Step, min(st1 * Step, vis), lane, M, L, y);
            rowOut(r, dst);
#pragma unroll
            for (int e = 0; e < D / 64; ++e) dst[lane + 64 * e] = !whole ? y[e] : L == 0.0f ? 0.0f : y[e] / L;
            if (lane == 0) rowSums(r, M, L);
        };
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            l[n] += __shfl_xor(l[n], 16);
            l[n] += __shfl_xor(l[n], 32);
        }
        if (KG == 1) {
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const int r = (rg * NR + n) * 16 + i;
                const float L = l[n] * kPInv;
                const float f = whole ? (L == 0.0f ? 0.0f : 1.0f / l[n]) : kPInv;
                float bad = L;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int v = 0; v < 4; ++v) bad = fmaf(o[n][d][v], 0.0f, bad);
                if (r < rows) {
                    float* dst;
                    rowOut(r, dst);
#pragma unroll
                    for (int d = 0; d < DT; ++d) *reinterpret_cast<f4a4*>(dst + 16 * d + 4 * g) = o[n][d] * f;
                    if (g == 0) rowSums(r, m[n], L);
                }
                unsigned long long lost = __ballot(r < rows && !(fabsf(bad) < INFINITY));
                lost |= lost >> 32;
                lost |= lost >> 16;
                if (__builtin_expect((lost & 0xFFFF) != 0, 0)) {
                    __threadfence();
                    for (unsigned left = (unsigned)lost & 0xFFFFu; left; left &= left - 1) again((rg * NR + n) * 16 + __builtin_ctz(left));
                }
            }
            if (u < u1) __syncthreads();
        } else if constexpr (KM > 1) {
            __syncthreads();
            float* jo = reinterpret_cast<float*>(lds);
            float* jm = jo + RT * G::ORow;  // (rt KG = RT)
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const int x = kg * rt + (rg * NR + n) * 16 + i;
#pragma unroll
                for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(jo + x * G::ORow + 16 * d + 4 * g) = o[n][d];
                if (g == 0) {
                    jm[2 * x] = m[n];
                    jm[2 * x + 1] = l[n];
                }
            }
            __syncthreads();
            constexpr int LP = D / 4;  // threads of a row (a wavefront, or a part of one)
            static_assert(NT % LP == 0 && LP <= 64);
            for (int r0 = 0; r0 < rows; r0 += NT / LP) {  // (the same for a wavefront's lanes but for the row)
                const int r = r0 + tid / LP, c = 4 * (tid % LP), rr = min(r, rows - 1);
                float M = -INFINITY, L = 0.0f;
                f32x4 y = zero;
                for (int w = 0; w < KG; ++w) M = fmaxf(M, jm[2 * (w * rt + rr)]);
                for (int w = 0; w < KG; ++w) {
                    const float mw = jm[2 * (w * rt + rr)], f = mw == -INFINITY ? 0.0f : ex2(mw - M);
                    const f32x4 ow = *reinterpret_cast<const f32x4*>(jo + (w * rt + rr) * G::ORow + c);
                    L = fmaf(f, jm[2 * (w * rt + rr) + 1], L);
                    y += f * ow;
                }
                float bad = L;
#pragma unroll
                for (int v = 0; v < 4; ++v) bad = fmaf(y[v], 0.0f, bad);
                const float f = whole ? (L == 0.0f ? 0.0f : 1.0f / L) : kPInv;
                if (r < rows) {
                    float* dst;
                    rowOut(r, dst);
                    *reinterpret_cast<f4a4*>(dst + c) = y * f;
                    if (c == 0) rowSums(r, M, L * kPInv);
                }
                const unsigned long long lost = __ballot(r < rows && !(fabsf(bad) < INFINITY));
                if (__builtin_expect(lost != 0, 0)) {
                    __threadfence();
                    for (int x = 0; x < 64 / LP; ++x)
                        if (LP == 64 ? lost != 0 : (lost >> (x * LP) & ((1ull << (LP & 63)) - 1)) != 0) again(r0 + wave * (64 / LP) + x);
                }
            }
            __syncthreads();
        }
    }
}

// The items that several workgroups had: o = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M). SG groups of a row's threads take the
// workgroups' sums in turn; their sums are added in order through LDS.
template <int D, int SG>
__global__ __launch_bounds__(256) void flash_pages_join_kernel(FpParams a, int rt) {
    constexpr int LP = D / 4, RB = 256 / LP / SG;
    __shared__ f32x4 sum[SG > 1 ? 256 : 1];
    __shared__ float2 ml[SG > 1 ? 256 / LP : 1];
    const int tid = threadIdx.x, c = 4 * (tid % LP), y = tid / LP, x = y / SG, sg = y % SG;
    const int item = blockIdx.x;
    const int total = a.head[0];
    const int* d = a.head + 4 + 8 * item;
    const int token0 = d[0], r0 = d[1], rows = d[2], kvh = d[3], w0 = d[4], n = d[5];
    if (item >= total || n <= 1) return;
    const long long stride = 2ll * rt * (D + 2);  // between workgroups; the first one's sum is its second, the others' their first
    const float* p0 = a.part + (long long)w0 * stride + rt * (D + 2);
    const float* pn = a.part + (long long)(w0 + 1) * stride;
    for (int b = blockIdx.y * RB; b < rows; b += gridDim.y * RB) {
        const int r = b + x, rr = min(r, rows - 1);
        float M = -INFINITY, L = 0.0f;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int Ahead = 4;
        for (int s0 = sg; s0 < n; s0 += SG * Ahead) {
            f32x4 z[Ahead];
            float ms[Ahead], ls[Ahead];
#pragma unroll
            for (int k = 0; k < Ahead; ++k) {
                const int s = min(s0 + SG * k, n - 1);
                const float* p = s == 0 ? p0 : pn + (s - 1) * stride;
                z[k] = *reinterpret_cast<const f4a4*>(p + rr * D + c);
                ms[k] = p[rt * D + 2 * rr];
                ls[k] = p[rt * D + 2 * rr + 1];
            }
#pragma unroll
            for (int k = 0; k < Ahead; ++k) {
                if (s0 + SG * k >= n) continue;
                const float top = fmaxf(M, ms[k]);  // (a NaN l comes with any m)
                const float f = M == -INFINITY ? 0.0f : ex2(M - top), h = ms[k] == -INFINITY ? 0.0f : ex2(ms[k] - top);
                L = ls[k] != ls[k] ? ls[k] : fmaf(h, ls[k], f * L);
                if (f != 1.0f) o = f == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o * f;
                if (h != 0.0f) o += h * z[k];
                M = top;
            }
        }
        if constexpr (SG > 1) {
            __syncthreads();  // (the last row's sums are read)
            sum[tid] = o;
            if (c == 0) ml[y] = make_float2(M, L);
            __syncthreads();
            float2 q[SG];
#pragma unroll
            for (int k = 0; k < SG; ++k) {
                q[k] = ml[y - sg + k];
                M = fmaxf(M, q[k].x);
            }
            L = 0.0f;
            o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < SG; ++k) {
                const float f = q[k].x == -INFINITY ? 0.0f : ex2(q[k].x - M);
                L = q[k].y != q[k].y ? q[k].y : fmaf(f, q[k].y, L);
                if (f != 0.0f) o += f * sum[tid + (k - sg) * LP];
            }
        }
        if (r >= rows || sg) continue;
        const int row = r0 + r, node = row / a.G, head = kvh * a.G + (row - node * a.G);
        const size_t at = (size_t)(token0 + node) * a.H + head;
        if (L != L) o = f32x4{NAN, NAN, NAN, NAN};
        *reinterpret_cast<f4a4*>(a.out + at * D + c) = L == 0.0f ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : o * (1.0f / L);
        if (a.lse && c == 0) a.lse[at] = L == 0.0f ? -INFINITY : fmaf(M, kLn2, logf(L));
    }
}

// How a call is launched: the form, workgroups (as many as run at once), rows of an item and the largest number of items.
struct FpPlan {
    int form, rt, groups, items, each;
    size_t bytes;
};
// Few rows, or little work: 16 rows to a wavefront (form 0); up to 128 rows of a sequence on average: 32 (1); more: eight wavefronts over the rows
// (2). The work is bounded by what the host knows, the tables' positions: a table with room for more than there is takes the form for more (tree of
// 24 nodes over 2050 positions: 19 us, with a table for 131072 25). us in calls back to back, 32 heads on 8, forms 0 / 1 / 2:
//   D = 128: 32 sequences of 4000 positions, 8 rows 104 / 107 / 109, 24 rows 117 / 112 / 109, 64 rows 161 / 129 / 123, 128 rows 315 / 189 / 183,
//   256 rows 612 / 308 / 302; the same, trees of 4 to 27 nodes on uneven lengths 229 / 154 / 178; one of 2000, 128 rows 20 / 23 / 28; 4 of 2000, 64
//   rows 25 / 30 / 29; one of 32000, 64 rows 57 / 55 / 54
//   D = 64, forms 0 / 1: 32 of 4000, 16 rows 62 / 60, 64 rows 89 / 75, 256 rows 288 / 222; one of 2000, 128 rows 18 / 21; 4 of 2000, 128 rows 23 / 31
//   D = 256 (registers for 16 rows, LDS for 64 positions), forms 1 / 2: 32 of 4000, 8 rows 190 / 191, 128 rows 347 / 340, 256 rows 690 / 657; one of 2000,
//   128 rows 25 / 34; 4 of 2000, 64 rows 44 / 37
FpPlan planOf(const kcFlashPagesDims& d) {
    FpPlan p{};
    const int64_t G = d.H / d.H_kv, rows = int64_t(d.N) * G, pairs = int64_t(d.N) * d.H * (int64_t(d.max_pages) * d.page);
    const int64_t each = d.seqs ? (rows + d.seqs - 1) / d.seqs : 0;
    const bool little = pairs <= (int64_t(1) << 37) / (d.D * d.D);
    if (d.D == 64) p.form = little || each <= 64 ? 0 : 1;
    else if (d.D == 128) p.form = little || each <= 16 ? 0 : each <= 128 ? 1 : 2;
    else p.form = each <= 128 ? 1 : 2;
    p.rt = (d.D == 256 ? 32 : 64) << p.form;
    p.groups = p.form == 1 || d.D == 64 ? 512 : 256;
    p.items = int((rows / p.rt + d.seqs) * d.H_kv);
    p.each = int(std::min<int64_t>(each, p.rt));
    p.bytes = 16 + size_t(p.items) * 32 + size_t(p.groups) * 2 * p.rt * (d.D + 2) * 4;
    return p;
}

template <int D, int NR, int W, int KM>
int run(FpParams p, const FpPlan& plan, hipStream_t s) {
    using G = FpGeo<D, NR, W, KM>;
    static const int ok = fromHip(hipFuncSetAttribute(reinterpret_cast<const void*>(flash_pages_kernel<D, NR, W, KM>),
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, G::Lds), "flash_pages: LDS size");
    if (ok) return ok;
    hipLaunchKernelGGL((flash_pages_kernel<D, NR, W, KM>), dim3(plan.groups), dim3(G::Threads), G::Lds, s, p);
    if (int e = fromHip(hipGetLastError(), "flash_pages")) return e;
    constexpr int Rows = 256 / (D / 4);
    // Many workgroups to an item, and not so many rows that there is a join workgroup for each CU anyway: several threads to a value. (us, 32 heads
    // on 8 of 128, with and without: one sequence of 20000 positions, 4 rows 27 / 31, 64 rows 44 / 52, 256 rows 77 / 75; 4 of 4000, 64 rows
    // 40 / 45, 256 rows 70 / 64; 8 of 4000, 64 rows 56 / 53.)
    if (plan.items * 8 <= plan.groups && plan.each <= 128) {
        hipLaunchKernelGGL((flash_pages_join_kernel<D, Rows>), dim3(plan.items, std::max(1, plan.each)), dim3(256), 0, s, p, G::RT);
    } else {
        hipLaunchKernelGGL((flash_pages_join_kernel<D, 1>), dim3(plan.items, (plan.each + Rows - 1) / Rows), dim3(256), 0, s, p, G::RT);
    }
    return fromHip(hipGetLastError(), "flash_pages (join)");
}

int runForm(int D, const FpParams& p, const FpPlan& plan, hipStream_t s) {
    switch (D + plan.form) {
        case 64: return run<64, 1, 4, 4>(p, plan, s);
        case 65: return run<64, 2, 4, 2>(p, plan, s);
        case 128: return run<128, 1, 4, 4>(p, plan, s);
        case 129: return run<128, 2, 4, 2>(p, plan, s);
        case 130: return run<128, 2, 8, 4>(p, plan, s);
        case 257: return run<256, 1, 4, 1>(p, plan, s);
        case 258: return run<256, 1, 8, 2>(p, plan, s);
        default: return fromHip(hipErrorInvalidValue, "flash_pages: form");
    }
}

}  // namespace

size_t flashPagesPartBytes(const kcFlashPagesDims& d) { return planOf(d).bytes; }

int launchFlashPages(const kcFlashPagesArgs& a, hipStream_t s) {
    const kcFlashPagesDims& d = a.d;
    if (d.N == 0 || d.seqs == 0) return 0;
    const FpPlan plan = planOf(d);
    FpParams p{};
    p.q = a.q;
    p.k = static_cast<const char*>(a.k);
    p.v = static_cast<const char*>(a.v);
    p.table = a.table;
    p.start = a.start;
    p.len = a.len;
    p.tree = a.tree;
    p.out = a.out;
    p.lse = a.lse;
    p.head = reinterpret_cast<int*>(a.part);
    p.part = a.part + 4 + 8 * (size_t)plan.items;
    p.k_row = d.k_row;
    p.k_head = d.k_head;
    p.v_row = d.v_row;
    p.v_head = d.v_head;
    p.H = d.H;
    p.H_kv = d.H_kv;
    p.G = d.H / d.H_kv;
    p.N = d.N;
    p.seqs = d.seqs;
    p.shift = __builtin_ctz((unsigned)d.page);
    p.max_pages = d.max_pages;
    p.n_pages = d.n_pages;
    p.tree_words = d.tree_words;
    p.q_tok = d.q_tok;
    p.q_head = d.q_head;
    p.table_row = d.table_row;
    p.groups = plan.groups;
    p.items = plan.items;
    p.scale = a.scale;
    return runForm(d.D, p, plan, s);
}

}  // namespace kcamd
