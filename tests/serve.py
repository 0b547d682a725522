"""Plain forms, in 64 bits, of the operators of a step of many requests over a paged cache, and the calls the tests make of the
kernels. Bounds on differences are derived beside each form."""
import math

import numpy as np

import kernelcore_amd as kc

GUARD = 0x5A5A5A5A


class Out:
    """An output of n values between guard words."""

    def __init__(self, n, dtype, fill=None):
        self.n, self.dtype = n, np.dtype(dtype)
        self.bytes = n * self.dtype.itemsize
        self.pad = (-self.bytes) % 4
        self.buf = kc.Buffer(256 + self.bytes + self.pad + 256)
        raw = np.full((512 + self.bytes + self.pad) // 4, GUARD, np.uint32)
        if fill is not None:
            raw.view(np.uint8)[256:256 + self.bytes] = np.ascontiguousarray(fill, self.dtype).reshape(-1).view(np.uint8)
        self.buf.upload(raw)
        self.ptr = self.buf.ptr + 256

    def get(self):
        raw = self.buf.download(np.uint8)
        assert (raw[:256].view(np.uint32) == GUARD).all(), "written before the output"
        assert (raw[256 + self.bytes + self.pad:].view(np.uint32) == GUARD).all(), "written behind the output"
        out = raw[256:256 + self.bytes].view(self.dtype).copy()
        self.buf.free()
        return out


def up(a, dtype):
    a = np.ascontiguousarray(a, dtype)
    return kc.Buffer.of(a) if a.nbytes else kc.Buffer(16)


# ---- kv_pages -----------------------------------------------------------------------------------------------------

def plain_pages(have, add, free, table, page, n_tokens, parent=None, words=0):
    """The definition, token by token. table: what the sequences' rows hold; returned as it is afterwards."""
    table = table.copy()
    seqs, max_pages = table.shape
    start, length, used = [0], [], 0
    slots, pos = np.full(n_tokens, -1, np.int64), np.zeros(n_tokens, np.int32)
    tree = np.zeros((n_tokens, words), np.uint32)
    for s in range(seqs):
        h, t0 = max(0, int(have[s])), start[-1]
        n = min(max(0, int(add[s])), n_tokens - t0)
        start.append(t0 + n)
        length.append(min(h + n, 2**31 - 1))
        for p in range(-(-h // page), min(max_pages, -(-(h + n) // page))):
            table[s, p] = free[used] if used < len(free) else -1
            used += 1
        seen, depth = [], []
        for i in range(n):
            p = h + i
            if p // page < max_pages and table[s, p // page] >= 0:
                slots[t0 + i] = int(table[s, p // page]) * page + p % page
            pos[t0 + i] = min(p, 2**31 - 1)
            if parent is not None:
                up_ = int(parent[t0 + i])
                if not 0 <= up_ < i:
                    up_ = -1
                seen.append((seen[up_] if up_ >= 0 else set()) | {i})
                depth.append(depth[up_] + 1 if up_ >= 0 else 0)
                pos[t0 + i] = min(h + depth[i], 2**31 - 1)
                for j in seen[i]:
                    if j < 32 * words:
                        tree[t0 + i, j >> 5] |= np.uint32(1 << (j & 31))
    return dict(start=np.array(start, np.int32), len=np.array(length, np.int32), slots=slots, pos=pos, used=np.array([used], np.int32),
                table=table, tree=tree.view(np.int32))


def run_pages(have, add, free, table, page, n_tokens, parent=None, words=0, row=None, stream=None):
    seqs, max_pages = table.shape
    row = max_pages if row is None else row
    wide = np.full((seqs, row), -77, np.int32)
    wide[:, :max_pages] = table
    bufs = dict(have=up(have, np.int32), add=up(add, np.int32), free=up(free, np.int32))
    if parent is not None:
        bufs["parent"] = up(parent, np.int32)
    o = dict(start=Out(seqs + 1, np.int32), len=Out(seqs, np.int32), slots=Out(n_tokens, np.int64), pos=Out(n_tokens, np.int32), used=Out(1, np.int32),
             table=Out(seqs * row, np.int32, wide), tree=Out(n_tokens * words, np.int32))
    kc.launch("kv_pages", kc.KvPagesArgs(**{k: b.ptr for k, b in bufs.items()}, **{k: x.ptr for k, x in o.items() if k != "tree" or words}, seqs=seqs,
                                         n_tokens=n_tokens, n_free=len(free), page=page, max_pages=max_pages, table_row=row, tree_words=words), stream)
    kc.synchronize()
    got = {k: x.get() for k, x in o.items()}
    got["table"] = got["table"].reshape(seqs, row)
    assert (got["table"][:, max_pages:] == -77).all()
    got["table"] = got["table"][:, :max_pages]
    got["tree"] = got["tree"].reshape(n_tokens, words)
    for b in bufs.values():
        b.free()
    return got


# ---- rope_ext -----------------------------------------------------------------------------------------------------

def plain_turn(x, pos, freqs, scale, n_rot, interleaved):
    """(values, bounds) of x [tokens][heads][D] turned. The angle is 2 pi of a fraction that was taken of a 64-bit product (off by 2^-53
    of the turns) and rounded to 32 bits (fraction at most 1/2: 2^-26 turns); cosine and sine within 4 units of 2^-24, times
    scale, two products and a sum, each rounded once more: for each of the pair's two terms the angle's error and 2^-21."""
    turns = pos.astype(np.longdouble)[:, None] * np.asarray(freqs, np.longdouble)
    a = ((turns - np.floor(turns)) * 2 * np.longdouble(np.pi)).astype(np.float64)
    c, s = np.cos(a)[:, None] * np.float64(np.float32(scale)), np.sin(a)[:, None] * np.float64(np.float32(scale))
    err = (2 * math.pi * (2.0 ** -26 + 2.0 ** -52 * np.abs(turns.astype(np.float64))) + 2.0 ** -21)[:, None] * abs(scale)
    y, b = x.astype(np.float64), np.zeros(x.shape)
    y = y.copy()
    i = np.arange(n_rot // 2)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + n_rot // 2)
    x0, x1 = x[..., lo].astype(np.float64), x[..., hi].astype(np.float64)
    y[..., lo], y[..., hi] = x0 * c - x1 * s, x0 * s + x1 * c
    b[..., lo] = b[..., hi] = err * (np.abs(x0) + np.abs(x1))
    return y, b


# ---- flash_pages_f16 ----------------------------------------------------------------------------------------------

class Pages:
    """One call: sequences with lens[s] positions of which the last nodes[s] are the step's tokens, in a shuffled paged cache. Tables
    have columns for `room` positions and rows of queries together at least (the kernel's form goes by what a table could hold)."""
    room = 0

    def __init__(self, H, K, D, lens, nodes, page=16, tree=True, words=2, scale=None, seed=0, spread=1.0, parent=None, spare=3):
        r = np.random.default_rng([seed, D, H, len(lens), page])
        self.H, self.K, self.D, self.page, self.words = H, K, D, page, words if tree else 0
        self.scale = 1.0 / math.sqrt(D) if scale is None else scale
        self.lens, self.nodes = np.asarray(lens, np.int64), np.asarray(nodes, np.int64)
        self.start = np.concatenate([[0], np.cumsum(self.nodes)]).astype(np.int32)
        self.N = int(self.start[-1])
        held = -(-self.lens // page)
        self.n_pages = int(held.sum()) + spare
        self.max_pages = max(1, int(held.max(initial=0)), -(-self.room // max(1, self.N * H) // page))
        order = r.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(lens), self.max_pages), -1, np.int32)
        at = 0
        for s, h in enumerate(held):
            self.table[s, :h] = order[at:at + h]
            at += h
        self.q = (r.standard_normal((self.N, H, D)) * spread).astype(np.float32)
        self.k, self.v = (r.standard_normal((self.n_pages * page, K, D)).astype(np.float16) for _ in range(2))
        # slots that hold no position: what may lie in memory
        used = np.zeros(self.n_pages * page, bool)
        for s in range(len(lens)):
            used[self.slots(s)] = True
        self.k[~used], self.v[~used] = np.nan, np.inf
        self.tree = None
        if tree:
            if parent is None:
                parent = np.concatenate([[-1 if i == 0 else int(r.integers(0, i)) for i in range(n)] for n in self.nodes] + [[]]).astype(np.int64)
            self.tree = plain_pages(np.zeros(len(lens)), self.nodes, [], np.zeros((len(lens), 1), np.int32), 16, self.N, parent, words)["tree"].view(np.uint32)

    def slots(self, s):
        p = np.arange(self.lens[s])
        return self.table[s, p // self.page].astype(np.int64) * self.page + p % self.page

    def seen(self, s):
        """[nodes][positions]"""
        n, T = int(self.nodes[s]), int(self.lens[s])
        j = np.arange(T) - (T - n)
        page = self.table[s, np.arange(T) // self.page]
        there = (page >= 0) & (page < self.n_pages)
        i = np.arange(n)[:, None]
        if self.tree is None:
            return (j[None] <= i) & there
        w = self.tree[self.start[s]:self.start[s + 1]]
        jj = np.clip(j, 0, 32 * self.words - 1)
        bit = (w[:, jj >> 5] >> (jj & 31).astype(np.uint32)[None] & 1) == 1
        return ((j < 0)[None] | (bit & (j >= 0) & (j < 32 * self.words))) & there

    def expected(self):
        """(out, bound on |difference|, lse, its bound). Scores: products of split q within 2^-21 of their terms, a walk of D f32
        additions, four more roundings; p in two fp16 parts, the second a multiple of 2^-24 of 2^11 p: 2^-36 of each value."""
        G = self.H // self.K
        out = np.zeros((self.N, self.H, self.D))
        bound = np.zeros_like(out)
        lse, lse_bound = np.full((self.N, self.H), -np.inf), np.zeros((self.N, self.H))
        for s in range(len(self.lens)):
            a, b, T = int(self.start[s]), int(self.start[s + 1]), int(self.lens[s])
            if a == b or T == 0:
                continue
            seen, slot = self.seen(s), np.clip(self.slots(s), 0, len(self.k) - 1)
            for h in range(self.H):
                k, v = self.k[slot, h // G].astype(np.float64), self.v[slot, h // G].astype(np.float64)
                q = self.q[a:b, h].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    x = np.where(seen, q @ k.T * np.float64(np.float32(self.scale)), -np.inf)
                    terms = np.where(seen, np.abs(q) @ np.abs(k.T) * abs(self.scale), 0.0)
                any_ = (seen & (x > -np.inf)).any(-1)
                top = np.where(any_, x.max(-1), 0.0)
                with np.errstate(invalid="ignore"):
                    p = np.where(seen, np.exp(x - top[:, None]), 0.0)
                total = np.where(any_, p.sum(-1), 1.0)
                w = p / total[:, None]
                safe = np.where(np.isfinite(v), v, 0.0)
                err = float(terms.max()) * (2.0 ** -21 + (math.sqrt(self.D) + 4) * 2.0 ** -24)
                out[a:b, h] = w @ safe
                bound[a:b, h] = (2 * err + 2.0 ** -20 + 4 * math.sqrt(T) * 2.0 ** -24) * (w @ np.abs(safe)) + 2.0 ** -36 * (seen.astype(float) @ np.abs(safe))
                lse[a:b, h] = np.where(any_, top + np.log(total), -np.inf)
                lse_bound[a:b, h] = err + 2.0 ** -20 + 4 * math.sqrt(T) * 2.0 ** -24 + 2.0 ** -22 * np.abs(np.where(any_, lse[a:b, h], 0.0))
        return out, bound, lse, lse_bound

    def dims(self, **over):
        hb = 2 * self.D
        d = dict(H=self.H, H_kv=self.K, D=self.D, N=self.N, seqs=len(self.lens), page=self.page, max_pages=self.max_pages, n_pages=self.n_pages,
                 tree_words=self.words, q_tok=self.H * self.D, q_head=self.D, table_row=self.max_pages, k_row=self.K * hb, k_head=hb,
                 v_row=self.K * hb, v_head=hb)
        d.update(over)
        return kc.FlashPagesDims(**d)

    def upload(self):
        b = dict(q=up(self.q, np.float32), k=up(self.k, np.float16), v=up(self.v, np.float16), table=up(self.table, np.int32),
                 start=up(self.start, np.int32), len=up(self.lens, np.int32))
        if self.tree is not None:
            b["tree"] = up(self.tree, np.uint32)
        return b

    def attend(self, stream=None, lse=True, extra=5):
        """(out, lse); `extra` rows behind the last sequence must stay as they were."""
        b = self.upload()
        b["q"].free()
        b["q"] = up(np.concatenate([self.q, np.full((extra, self.H, self.D), np.nan, np.float32)]), np.float32)
        if self.tree is not None:
            b["tree"].free()
            b["tree"] = up(np.concatenate([self.tree, np.full((extra, self.words), 0xFFFFFFFF, np.uint32)]), np.uint32)
        d = self.dims(N=self.N + extra)
        n = self.N + extra
        part = Out(kc.flash_pages_part_bytes(d), np.uint8, np.full(kc.flash_pages_part_bytes(d), 0xFF, np.uint8))
        out, sums = Out(n * self.H * self.D, np.float32, np.full(n * self.H * self.D, 7.0)), Out(n * self.H, np.float32, np.full(n * self.H, 7.0))
        kc.launch("flash_pages_f16", kc.FlashPagesArgs(**{k: x.ptr for k, x in b.items()}, out=out.ptr, lse=sums.ptr if lse else None, part=part.ptr, d=d,
                                                       scale=self.scale), stream)
        kc.synchronize()
        part.get()
        o, s = out.get().reshape(n, self.H, self.D), sums.get().reshape(n, self.H)
        for x in b.values():
            x.free()
        assert (o[self.N:] == 7).all() and (s[self.N:] == 7).all()
        return o[:self.N], s[:self.N]

    def check(self):
        out, sums = self.attend()
        want, bound, lse, lse_bound = self.expected()
        bad = ~(np.abs(out - want) <= bound)
        assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.abs(out - want)[bad].max()), float(bound[bad].min()))
        fin = np.isfinite(lse)
        assert (np.isneginf(sums) == ~fin).all()
        assert (np.abs(sums[fin] - lse[fin]) <= lse_bound[fin]).all()
        assert (out[~fin] == 0).all()
        return out, sums


# ---- sample_rows --------------------------------------------------------------------------------------------------

def plain_sample(l, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens that are right, their probabilities): the token of the definition, and any other that a border moved by 2^-40 of the
    whole would give (weights of 2^-52 and steps of 2^-43 of the largest weight, up to 2^20 of them; a difference of cumulated
    weights beside a border of that size is not what is tested)."""
    l = np.asarray(l, np.float32)
    if np.isnan(l).any() or np.isposinf(l).any() or np.isneginf(l).all():
        return [-1], [0.0]
    order = np.argsort(-l.astype(np.float64), kind="stable")
    if not temperature > 0:
        return [int(order[0])], [1.0]
    z = l[order].astype(np.longdouble) / np.longdouble(np.float32(temperature))
    w = np.where(np.isneginf(l[order]), np.longdouble(0), np.exp(np.where(np.isneginf(l[order]), 0, z - z[0])))
    finite = int(np.isfinite(l).sum())
    eps = np.longdouble(2.0 ** -40)
    k = min(top_k, finite) if top_k > 0 else finite
    c = np.cumsum(w)

    def cuts(e):
        m = k
        if top_p < 1:
            m = min(m, int((c[:k] < np.longdouble(np.float32(top_p)) * c[k - 1] * (1 + e)).sum()) + 1) if top_p > 0 else 1
        if min_p > 0:
            m = min(m, max(1, int((w >= np.longdouble(np.float32(min_p)) * (1 + e)).sum())))
        return max(m, 1)
    tokens, probs = [], []
    uu = np.longdouble(0) if not u > 0 else np.longdouble(np.float32(u))
    for m in sorted({cuts(0), cuts(eps), cuts(-eps)}):
        last = int(np.flatnonzero(w[:m] > 0)[-1])
        for e in (0, eps, -eps):
            i = min(last, int((c[:m] <= uu * c[m - 1] + e * c[m - 1]).sum()))
            if int(order[i]) not in tokens:
                tokens.append(int(order[i]))
                probs.append(float(w[i] / c[m - 1]))
    return tokens, probs


def run_sample(l, u, temperature=None, top_k=None, top_p=None, min_p=None, row=None, stream=None, probs=True):
    l = np.asarray(l, np.float32)
    R, V = l.shape
    row = V if row is None else row
    wide = np.full((R, row), np.nan, np.float32)
    wide[:, :V] = l
    ins = dict(logits=up(wide, np.float32), u=up(u, np.float32))
    for name, x, t in (("temperature", temperature, np.float32), ("top_k", top_k, np.int32), ("top_p", top_p, np.float32), ("min_p", min_p, np.float32)):
        if x is not None:
            ins[name] = up(np.broadcast_to(np.asarray(x, t), R), t)
    n = kc.sample_rows_part_bytes(R, V)
    part, tokens, pr = Out(n, np.uint8, np.full(n, 0xFF, np.uint8)), Out(R, np.int32), Out(R, np.float32)
    kc.launch("sample_rows", kc.SampleRowsArgs(**{k: b.ptr for k, b in ins.items()}, tokens=tokens.ptr, probs=pr.ptr if probs else None, part=part.ptr,
                                               row=row, rows=R, n_vocab=V), stream)
    kc.synchronize()
    part.get()
    for b in ins.values():
        b.free()
    return tokens.get(), pr.get()
