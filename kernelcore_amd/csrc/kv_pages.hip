// kv_pages.hip -- kv_pages: pages, slots, positions and tree masks of the tokens that a step adds to a paged cache.
//
// start = prefix sums of the counts, page offsets = prefix sums of the new pages; a token's page is an entry of its sequence's table
// row where the page was there before, else the next of the free list (which the table is given by the token at the page's
// foot: every new page begins at a token of the step). So no token waits for what another workgroup writes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "internal.hpp"
#include "kserve.hpp"

namespace kcamd {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64, kPer = 4;  // sequences of a thread in a round
// Tokens of a launch where there are trees: a token's walk up its tree ends with the launch's first one, and goes on from what the launch
// before wrote. (130 ns a node, so that a launch takes 35 ms at most; without this end a longer chain's time grew without bound. Launches of 32768
// would cost a step of many short trees more than they save: 20000 trees of 5 nodes 125 us for 40.)
constexpr int kLaunch = 1 << 18;

struct PagesArgs {
    const int *have, *add, *free, *parent;
    int* table;
    int *start, *len;
    long long* slots;
    int *pos, *used, *tree;
    int seqs, n_tokens, n_free, shift, max_pages, table_row, tree_words;
    int t0, end;  // the launch's tokens
};

// The sums of x over the threads before this one (all: over all of them).
__device__ __forceinline__ int sumBefore(int x, int* waves, int tid, int& all) {
    const int lane = tid & 63, wave = tid >> 6;
    int y = x;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int z = __shfl_up(y, o);
        if (lane >= o) y += z;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = y;
    __syncthreads();
    all = 0;
    int before = y - x;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? waves[w] : 0;
        all += waves[w];
    }
    return before;
}

// A workgroup: 256 tokens. It sums over the sequences by itself (1024 in a round, until its tokens are covered): what other workgroups
// found would take a launch of its own. Latency bounds it: 8 requests of a token 4 us, 256 of 97 tokens 4.2, 500 trees of 24 nodes
// 5.0 (their longest chain of parents, from LDS). Each token walks up its tree by itself, a load for each ancestor: a prompt of 2048 tokens that is
// given as a chain among trees takes 360 us.
__global__ __launch_bounds__(kThreads) void kv_pages_kernel(PagesArgs a) {
    __shared__ int waves[2][kWaves];
    __shared__ int first[kThreads];                             // a token that is its sequence's first here: its number, else 0
    __shared__ int4 rec[kThreads];                              // its sequence: number, start, have, pages taken before it
    __shared__ int parents[2 * kThreads];
    __shared__ int last[kWaves];
    const int tid = threadIdx.x, t0 = a.t0 + blockIdx.x * kThreads, t = t0 + tid;
    const int per = 1 << a.shift;
    int above[2] = {-1, -1};  // the parents of this token and of the one 256 before it, for LDS once the sums are done
    if (a.parent && a.n_tokens > 0) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int at = t + kThreads * (k - 1), x = a.parent[min(max(at, 0), a.n_tokens - 1)];
            above[k] = at >= 0 && at < a.n_tokens ? x : -1;
        }
    }
    first[tid] = 0;
    int tokens = 0, pages = 0;  // before the round's sequences
    for (int s0 = 0; s0 < a.seqs; s0 += kPer * kThreads) {
        if (t0 && tokens >= t0 + kThreads) break;  // (the first workgroup writes the sequences' numbers)
        int have[kPer], add[kPer], need[kPer], sum = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const int s = s0 + kPer * tid + e, at = min(s, a.seqs - 1);  // (loads without conditions are under way together)
            have[e] = max(a.have[at], 0);
            add[e] = min(max(a.add[at], 0), a.n_tokens);
            have[e] = s < a.seqs ? have[e] : 0;
            // (a sequence brings no more than n_tokens, and a thread's four stay below 2^31 together)
            add[e] = s < a.seqs ? add[e] : 0;
            sum = (int)min((long long)sum + add[e], (long long)a.n_tokens);
        }
        // (sums that stay below 2^31: past n_tokens they only have to stay past it)
        __syncthreads();
        int before;
        {
            const int lane = tid & 63, wave = tid >> 6;
            long long y = sum;
#pragma unroll
            for (int o = 1; o < 64; o *= 2) {
                const long long z = __shfl_up(y, o);
                if (lane >= o) y += z;
            }
            if (lane == 63) waves[0][wave] = (int)min(y, (long long)a.n_tokens);
            __syncthreads();
            long long b = y - sum + tokens, all = tokens;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                b += w < wave ? waves[0][w] : 0;
                all += waves[0][w];
            }
            before = (int)min(b, (long long)a.n_tokens);
            tokens = (int)min(all, (long long)a.n_tokens);
        }
        int at[kPer], pagesHere = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            at[e] = before;
            add[e] = min(add[e], a.n_tokens - before);
            before += add[e];
            const long long end = (long long)have[e] + add[e];
            const long long p0 = ((long long)have[e] + per - 1) >> a.shift, p1 = (end + per - 1) >> a.shift;
            need[e] = (int)(min(p1, (long long)a.max_pages) - min(p0, (long long)a.max_pages));
            pagesHere += need[e];
        }
        int allPages;
        int pb = pages + sumBefore(pagesHere, waves[1], tid, allPages);
        pages += allPages;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const int s = s0 + kPer * tid + e;
            if (s < a.seqs) {
                if (add[e] > 0 && at[e] < t0 + kThreads && at[e] + add[e] > t0) {
                    const int x = max(at[e], t0) - t0;
                    first[x] = x + 1;
                    rec[x] = int4{s, at[e], have[e], pb};
                }
                if (t0 == 0) {
                    a.start[s] = at[e];
                    a.len[s] = (int)min((long long)have[e] + add[e], (long long)INT_MAX);
                }
            }
            pb += need[e];
        }
    }
    parents[tid] = above[0];
    parents[tid + kThreads] = above[1];
    if (t0 == 0 && tid == 0) {
        a.start[a.seqs] = tokens;
        a.used[0] = pages;
    }
    __syncthreads();
    // the last token before this one, or this one, that is its sequence's first here
    int x = first[tid];
    {
        const int lane = tid & 63, wave = tid >> 6;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int z = __shfl_up(x, o);
            if (lane >= o) x = max(x, z);
        }
        if (lane == 63) last[wave] = x;
        __syncthreads();
        for (int w = 0; w < wave; ++w) x = max(x, last[w]);
    }
    if (t >= a.end) return;
    int* words = a.tree ? a.tree + (size_t)t * a.tree_words : nullptr;
    if (t >= tokens || x == 0) {  // (behind the last sequence; tokens is short only in workgroups that others' tokens end)
        a.slots[t] = -1;
        if (a.pos) a.pos[t] = 0;
        for (int w = 0; w < a.tree_words; ++w) words[w] = 0;
        return;
    }
    const int4 r = rec[x - 1];
    const int node = t - r.y;
    const long long p = (long long)r.z + node, pi = p >> a.shift, held = ((long long)r.z + per - 1) >> a.shift;
    int page = -1;
    if (pi < a.max_pages) {
        int* entry = a.table + (size_t)r.x * a.table_row + pi;
        if (pi < held) {
            page = *entry;
        } else {
            const long long f = r.w + (pi - held);
            page = f < a.n_free ? a.free[f] : -1;
            if ((p & (per - 1)) == 0) *entry = page;
        }
    }
    a.slots[t] = page < 0 ? -1ll : ((long long)page << a.shift) + (p & (per - 1));
    int depth = node;
    if (a.parent && a.tree_words <= 2 && r.y >= t0 - kThreads) {
        // up to 64 bits, all parents in LDS: the bits in registers (500 trees of 24 nodes: 0.8 us less than by the form below)
        const int* up = parents + (r.y - (t0 - kThreads));
        unsigned long long bits = 0;
        depth = -1;
        int next = node, cur;
        do {
            cur = next;
            bits |= cur < 64 ? 1ull << cur : 0;
            ++depth;
            next = up[cur];
        } while ((unsigned)next < (unsigned)cur);
        words[0] = (int)bits;
        if (a.tree_words == 2) words[1] = (int)(bits >> 32);
    } else if (a.parent) {
        // the node and its ancestors, numbers descending: a word is written when the next one begins
        depth = 0;
        int w = a.tree_words - 1;
        uint32_t bits = 0;
        int cur = node;
        const unsigned least = max(a.t0 - r.y, 0);  // the sequence's first node of this launch
        while (true) {
            if (cur < 32 * a.tree_words) {
                for (; w > cur >> 5; --w, bits = 0) words[w] = (int)bits;
                bits |= 1u << (cur & 31);
            }
            const int k = r.y + cur - (t0 - kThreads);
            const int up = k >= 0 ? parents[k] : a.parent[r.y + cur];
            if (up - least >= cur - least) break;
            cur = up;
            ++depth;
        }
        const int up = least ? a.parent[r.y + cur] : -1;
        if (up >= 0 && up < cur) {
            // (an ancestor of the launch before: its words and its position)
            const int* others = a.tree + (size_t)(r.y + up) * a.tree_words;
            for (; w >= 0; --w, bits = 0) words[w] = (int)bits | others[w];
            if (a.pos) a.pos[t] = (int)min((long long)a.pos[r.y + up] + depth + 1, (long long)INT_MAX);
            return;
        }
        for (; w >= 0; --w, bits = 0) words[w] = (int)bits;
    }
    if (a.pos) a.pos[t] = (int)min((long long)r.z + depth, (long long)INT_MAX);
}

}  // namespace

int launchKvPages(const kcKvPagesArgs& a, hipStream_t s) {
    PagesArgs p{a.have, a.add, a.free, a.parent, a.table, a.start, a.len, reinterpret_cast<long long*>(a.slots), a.pos, a.used,
                a.tree, a.seqs, a.n_tokens, a.n_free, __builtin_ctz((unsigned)a.page), a.max_pages, a.table_row, a.tree ? a.tree_words : 0, 0, 0};
    do {
        const int n = a.parent ? std::min(kLaunch, a.n_tokens - p.t0) : a.n_tokens;
        p.end = p.t0 + n;
        hipLaunchKernelGGL(kv_pages_kernel, dim3(n > 0 ? (n - 1) / kThreads + 1 : 1), dim3(kThreads), 0, s, p);
        if (int e = fromHip(hipGetLastError(), "kv_pages")) return e;
        p.t0 = p.end;
    } while (p.t0 < a.n_tokens);
    return 0;
}

}  // namespace kcamd
