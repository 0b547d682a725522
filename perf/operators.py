"""The serving operators over a key/value cache, as measurable cases: storing rows as 4-bit blocks and reading them
back, attention over an fp16 or a 4-bit cache with shaped scores (a tanh cap, a bias by distance, documents, a
prefix), the accumulated attention weight of every cached position, and the choice and compaction of the positions
to keep.

Head counts and widths are the repository's own (32 or 24 query heads of 128 over 8 KV heads) or generic. Queries, keys
and values are N(0, 1), as after their norms and rotation. Everything is made here from the seed with torch.

`run` gives each operator's plain form in elementary torch operations where `own` is false, and the library's kernels
where it is true."""
import math

import numpy as np
import torch

own = False


# ---- the cases --------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token's key row (8 heads of 128) stored into the cache of a layer and read back: latency alone
        dict(name="store_token", kind="store", rows=1, n=1024, cache=4096),
        # a ragged prompt's key rows at scattered cache slots
        dict(name="store_prompt_1777", kind="store", rows=1777, n=1024, cache=4096),
        # a decoded token's attention over a conversation held in 4 bits
        dict(name="q4_token_8k", kind="attend", cache="q4_0", heads=32, heads_kv=8, dim=128, tokens=1, ctx=8191, causal=True,
             prefix=0, docs=0, cap=0.0, bias=False, dense=False, kept=False, lse=False),
        # the same over the longest context, where a 4-bit cache is what fits
        dict(name="q4_token_128k", kind="attend", cache="q4_0", heads=32, heads_kv=8, dim=128, tokens=1, ctx=131072, causal=True,
             prefix=0, docs=0, cap=0.0, bias=False, dense=False, kept=False, lse=False),
        # a ragged chunk of a prompt behind earlier ones
        dict(name="q4_chunk_1000", kind="attend", cache="q4_0", heads=32, heads_kv=8, dim=128, tokens=1000, ctx=3577, causal=True,
             prefix=0, docs=0, cap=0.0, bias=False, dense=False, kept=False, lse=False),
        # a few drafted tokens checked at once, scores capped; the sums kept for the weights of the cached positions
        dict(name="f16_draft_capped", kind="attend", cache="f16", heads=24, heads_kv=8, dim=128, tokens=5, ctx=2049, causal=True,
             prefix=0, docs=0, cap=30.0, bias=False, dense=False, kept=False, lse=True),
        # a prompt with a bidirectional prefix (an image, an instruction) and a bias by distance
        dict(name="f16_prefix_bias", kind="attend", cache="f16", heads=24, heads_kv=8, dim=128, tokens=2048, ctx=2048, causal=True,
             prefix=300, docs=0, cap=0.0, bias=True, dense=False, kept=False, lse=False),
        # many prompts packed into one batch, none seeing another, scores capped: the largest
        dict(name="f16_packed_documents", kind="attend", cache="f16", heads=32, heads_kv=8, dim=128, tokens=4096, ctx=4096,
             causal=True, prefix=0, docs=11, cap=50.0, bias=False, dense=False, kept=False, lse=False),
        # what a prompt's last tokens looked at, before the cache is thinned
        dict(name="weights_window_64", kind="weights", cache="q4_0", heads=32, heads_kv=8, dim=128, tokens=64, ctx=8192, causal=True,
             prefix=0, docs=0, cap=0.0, bias=False, dense=False, kept=False),
        # the same after each decoded token, over a cache that was thinned before
        dict(name="weights_token", kind="weights", cache="f16", heads=24, heads_kv=8, dim=128, tokens=1, ctx=4099, causal=True,
             prefix=0, docs=0, cap=0.0, bias=False, dense=False, kept=True),
        # a long context cut to a quarter
        dict(name="evict_16k", kind="evict", heads_kv=8, dim=128, ctx=16384, keep=4096, first=4, recent=256),
        # a small cache at its budget
        dict(name="evict_1500", kind="evict", heads_kv=8, dim=128, ctx=1500, keep=1024, first=4, recent=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "attend", "weights", "weights", "evict"])
    if kind == "store":
        cache = _log(rng, 64, 32768)
        return dict(kind=kind, rows=_log(rng, 1, min(cache, 4096)), n=32 * _log(rng, 2, 64), cache=cache)
    if kind == "evict":
        ctx = _log(rng, 33, 65536)
        keep = max(8, int(ctx * rng.uniform(0.1, 1.0)))
        first = rng.choice([0, 1, 4])
        return dict(kind=kind, heads_kv=rng.choice([1, 2, 8]), dim=rng.choice([64, 128, 256]), ctx=ctx, keep=keep, first=first,
                    recent=rng.randint(0, keep - first))
    heads, heads_kv = rng.choice([(32, 8), (32, 8), (24, 8), (8, 8), (16, 1), (10, 2)])
    dim = rng.choice([64, 128, 128, 256])
    if kind == "weights":
        tokens = rng.choice([1, _log(rng, 1, 256)])
    else:
        tokens = rng.choice([1, rng.randint(1, 8), _log(rng, 9, 2048)])
    # (a pass's plain form holds tokens * heads * ctx scores)
    room = min(131072, (1 << 28) // (tokens * heads) * 128 // dim)
    ctx = _log(rng, tokens, max(tokens, room))
    shaped = rng.random() < 0.6
    dense = shaped and rng.random() < 0.25
    docs = 0 if not shaped or dense or rng.random() < 0.6 else min(ctx, rng.randint(2, 16))
    c = dict(kind=kind, cache=rng.choice(["q4_0", "f16"]), heads=heads, heads_kv=heads_kv, dim=dim, tokens=tokens, ctx=ctx,
             causal=not dense and rng.random() < 0.85, prefix=rng.randint(0, ctx) if shaped and rng.random() < 0.3 else 0, docs=docs,
             cap=rng.choice([0.0, 20.0, 50.0]) if shaped else 0.0, bias=shaped and rng.random() < 0.4, dense=dense,
             kept=not docs and rng.random() < 0.2)
    if kind == "attend":
        c["lse"] = rng.random() < 0.3
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------

def _gen(seed, *ids):
    for i in ids:
        seed = (seed * 1000003 + i + 7) & 0x7FFFFFFFFFFF
    return torch.Generator(device="cuda").manual_seed(seed & 0x7FFFFFFFFFFF)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _q4_cache(g, rows, heads, dim):
    """rows x heads x dim values as 4-bit blocks: uint8 [rows, heads, dim / 32 * 18] (a block of 32 values: an fp16 scale d,
    then 16 bytes; byte e holds the code of value e in its low four bits and that of value e + 16 in its high ones; a
    code c stands for d (c - 8))."""
    out = torch.empty(rows, heads, dim // 32, 18, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (heads * dim))
    for r0 in range(0, rows, step):
        r1 = min(rows, r0 + step)
        x = _normal(g, r1 - r0, heads, dim // 32, 32)
        d = x.abs().amax(-1, keepdim=True) / 8
        c = (x / d + 8.5).floor().clamp(0, 15).to(torch.uint8)
        out[r0:r1, ..., :2] = d.half().view(torch.uint8)
        out[r0:r1, ..., 2:] = c[..., :16] | (c[..., 16:] << 4)
    return out.view(rows, heads, dim // 32 * 18)


def _documents(ctx, docs):
    """Document numbers of ctx packed positions: lengths as 1 : 2 : ... : docs."""
    ends = np.rint(np.cumsum(np.arange(1, docs + 1)) / (docs * (docs + 1) / 2) * ctx).astype(np.int64)
    return np.searchsorted(ends, np.arange(ctx), side="right")


def _slopes(heads):
    return torch.exp2(-8.0 * torch.arange(1, heads + 1, dtype=torch.float32) / heads)


def _attention_inputs(c, seed):
    H, K, D, N, T = c["heads"], c["heads_kv"], c["dim"], c["tokens"], c["ctx"]
    t = dict(q=_normal(_gen(seed, 1), N, H, D))
    if c["cache"] == "f16":
        t["k"], t["v"] = _normal(_gen(seed, 2), T, K, D).half(), _normal(_gen(seed, 3), T, K, D).half()
    else:
        t["k"], t["v"] = _q4_cache(_gen(seed, 2), T, K, D), _q4_cache(_gen(seed, 3), T, K, D)
    first = T - N
    if c["kept"]:  # the positions that earlier evictions left in each head's cache: ascending, the queries' own last
        gaps = torch.randint(1, 4, (K, T), generator=_gen(seed, 4), device="cuda")
        gaps[:, max(first, 0):] = 1
        pos = gaps.cumsum(1)
        t["kpos"] = (pos + (pos[:, -1].max() - pos[:, -1:])).int().contiguous()
        first = int(t["kpos"][0, -1]) - N + 1
    t["qpos"] = torch.arange(first, first + N, dtype=torch.int32, device="cuda")
    if c["docs"]:
        ids = torch.from_numpy(_documents(T, c["docs"])).int().cuda()
        t["kdoc"], t["qdoc"] = ids, ids[T - N:].contiguous()
    if c["bias"]:
        t["slopes"] = _slopes(H).cuda()
    if c["dense"]:  # what a program adds to the scores itself: some places -inf, some a bias
        m = _normal(_gen(seed, 5), N, T).half()
        m[torch.rand(N, T, generator=_gen(seed, 6), device="cuda") < 0.5] = -math.inf
        pad = torch.full((N, (T + 1) // 2 * 2 - T), -math.inf, dtype=torch.float16, device="cuda")
        t["mask"] = torch.cat([m, pad], 1).contiguous()
    return t


def prepare(case, seed):
    c = dict(case)
    if c["kind"] == "store":
        g = _gen(seed, 1)
        t = dict(src=_normal(g, c["rows"], c["n"]),
                 idx=torch.randperm(c["cache"], generator=g, device="cuda")[:c["rows"]].contiguous(),
                 cache=torch.zeros(c["cache"], c["n"] // 32 * 18, dtype=torch.uint8, device="cuda"))
    elif c["kind"] == "evict":
        K, D, T = c["heads_kv"], c["dim"], c["ctx"]
        t = dict(k=_normal(_gen(seed, 2), T, K, D).half(), v=_normal(_gen(seed, 3), T, K, D).half(),
                 w=torch.rand(K, T, generator=_gen(seed, 4), device="cuda") ** 8,
                 kpos=torch.arange(T, dtype=torch.int32, device="cuda").repeat(K, 1))
    else:
        t = _attention_inputs(c, seed)
        if c["kind"] == "weights":
            t["lse"] = _sums64(c, t).float()
            t["w_in"] = torch.rand(c["heads_kv"], c["ctx"], generator=_gen(seed, 8), device="cuda")
    s = dict(case=c, **t)
    if own:
        _own_state(s)
    torch.cuda.synchronize()
    return s


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


# ---- the plain forms --------------------------------------------------------------------------------------------

def _plain_store(s):
    # (in 64 bits: which of two codes a value next to their border gets)
    x = s["src"].view(s["src"].shape[0], -1, 32).double()
    a = x.abs()
    top = a.amax(-1, keepdim=True)
    at = torch.where(a == top, torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
    d = x.gather(-1, at) / -8
    c = torch.where(d == 0, 8.0, (x / d + 8.5).floor().clamp(0, 15)).to(torch.uint8)
    blocks = torch.cat([d.float().half().view(torch.uint8), c[..., :16] | (c[..., 16:] << 4)], -1)
    s["cache"][s["idx"]] = blocks.view(blocks.shape[0], -1)
    return _plain_q4(s["cache"][s["idx"]])


def _plain_q4(b):
    """The values that rows of 4-bit blocks stand for: [..., n / 32 * 18] bytes -> [..., n] f32."""
    b = b.view(*b.shape[:-1], -1, 18)
    d = b[..., :2].contiguous().view(torch.float16).float()
    c = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).float() - 8
    return (d * c).flatten(-2)


def _plain_scores(s):
    """The shaped scores, masked places -inf: [KV heads, heads / KV heads * tokens, positions], f32."""
    c = s["case"]
    H, K, D, N, T = c["heads"], c["heads_kv"], c["dim"], c["tokens"], c["ctx"]
    k = s["k"].float() if c["cache"] == "f16" else _plain_q4(s["k"])
    q = s["q"].view(N, K, H // K, D).permute(1, 2, 0, 3).reshape(K, -1, D)
    x = torch.matmul(q, k.permute(1, 2, 0)) * (1.0 / math.sqrt(D))
    x = x.view(K, H // K, N, T)
    if c["cap"]:
        x = torch.tanh(x / c["cap"]) * c["cap"]
    kpos = s["kpos"] if c["kept"] else torch.arange(T, device=q.device)[None]
    kpos, qpos = kpos[:, None, None, :], s["qpos"][:, None]
    if c["bias"]:
        x = x - s["slopes"].view(K, H // K, 1, 1) * (qpos - kpos).abs().float()
    if c["dense"]:
        x = x + s["mask"][:, :T].float()
    if c["causal"]:
        x = x.masked_fill((kpos > qpos) & (kpos >= c["prefix"]), -math.inf)
    if c["docs"]:
        x = x.masked_fill(s["qdoc"][:, None] != s["kdoc"][None], -math.inf)
    return x.view(K, -1, T)


def _plain_attend(s):
    c = s["case"]
    H, K, D, N = c["heads"], c["heads_kv"], c["dim"], c["tokens"]
    v = s["v"].float() if c["cache"] == "f16" else _plain_q4(s["v"])
    x = _plain_scores(s)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(1, 0, 2)) / torch.where(total == 0, 1.0, total)
    o = o.view(K, H // K, N, D).permute(2, 0, 1, 3).reshape(N, H, D)
    if not c["lse"]:
        return o
    return o, (top + torch.log(total)).view(H, N).t().contiguous()


def _plain_weights(s):
    c = s["case"]
    K = c["heads_kv"]
    lse = s["lse"].t().reshape(K, -1, 1)
    p = torch.exp(_plain_scores(s) - torch.where(lse == -math.inf, 0.0, lse))
    return 0.9 * s["w_in"] + p.sum(1)


def _plain_evict(s):
    c = s["case"]
    T, n, first, recent = c["ctx"], c["keep"], c["first"], c["recent"]
    w = s["w"].clone()
    w[:, :first] = math.inf
    w[:, T - recent:] = math.inf
    keep = torch.sort(w, dim=1, descending=True, stable=True)[1][:, :n].sort(1)[0]  # (ties: the lowest index)
    rows = keep.t()[:, :, None].expand(-1, -1, c["dim"])
    return keep.int(), s["k"].gather(0, rows), s["v"].gather(0, rows), s["w"].gather(1, keep), s["kpos"].gather(1, keep)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------

def _values64(c, x):
    """A cache's values: [positions, KV heads, dim]."""
    if c["cache"] == "f16":
        return x.double()
    b = x.view(x.shape[0], x.shape[1], -1, 18)
    out = torch.empty(*b.shape[:3], 32, dtype=torch.float64, device=x.device)
    lo, hi = b[..., 2:].remainder(16), b[..., 2:].div(16, rounding_mode="floor")
    out[..., :16], out[..., 16:] = lo.double() - 8, hi.double() - 8
    return (out * b[..., :2].contiguous().view(torch.float16).double()).reshape(x.shape[0], x.shape[1], -1)


def _head64(c, t, h, keys):
    """Scores of query head h against its keys: [tokens, positions]; -inf where the key is not seen."""
    g = h // (c["heads"] // c["heads_kv"])
    x = t["q"][:, h].double() @ keys[:, g].t() / math.sqrt(c["dim"])
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    i = t["qpos"].double()[:, None]
    j = (t["kpos"][g] if c["kept"] else torch.arange(c["ctx"], device=x.device)).double()[None]
    if c["bias"]:
        x = x - 2.0 ** (-8.0 * (h + 1) / c["heads"]) * (i - j).abs()
    if c["dense"]:
        x = x + t["mask"][:, :c["ctx"]].double()
    seen = torch.ones_like(x, dtype=torch.bool)
    if c["causal"]:
        seen &= (j <= i) | (j < c["prefix"])
    if c["docs"]:
        seen &= t["qdoc"][:, None] == t["kdoc"][None]
    return torch.where(seen, x, -math.inf)


def _sums64(c, t):
    """log sum exp of the scores: [tokens, heads]."""
    keys = _values64(c, t["k"])
    return torch.stack([torch.logsumexp(_head64(c, t, h, keys), 1) for h in range(c["heads"])], 1)


def exact(case, seed):
    c = dict(case)
    if c["kind"] == "evict":
        out = _plain_evict(prepare(case, seed))  # (values moved, none computed)
        return [None, out[1].double(), out[2].double(), out[3].double(), None]
    t = prepare(case, seed)
    if c["kind"] == "store":
        x = t["src"].view(c["rows"], -1, 32).double()
        far = x.abs().argmax(-1, keepdim=True)
        d = -x.gather(-1, far) / 8
        step, y = d.abs(), x * d.sign()
        code = sum(((k - 8.5) * step <= y).double() for k in range(1, 16))
        return (torch.where(step == 0, 0.0, code - 8) * d.float().half().double()).view(c["rows"], -1)
    keys, values = _values64(c, t["k"]), _values64(c, t["v"])
    G = c["heads"] // c["heads_kv"]
    o, sums, w = [], [], 0.9 * t["w_in"].double() if c["kind"] == "weights" else None
    for h in range(c["heads"]):
        x = _head64(c, t, h, keys)
        z = torch.logsumexp(x, 1, keepdim=True) if w is None else t["lse"][:, h, None].double()
        p = torch.where(z == -math.inf, 0.0, torch.exp(x - z))
        if w is None:
            o.append(p @ values[:, h // G])
            sums.append(z[:, 0])
        else:
            w[h // G] += p.sum(0)
    if w is not None:
        return w
    o = torch.stack(o, 1)
    return (o, torch.stack(sums, 1)) if c["lse"] else o


# ---- the library's kernels --------------------------------------------------------------------------------------

_LIB = {}


def _lib():
    """The package and a stream of the library's."""
    if not _LIB:
        import ctypes

        import kernelcore_amd as kc
        kc.init()
        s = ctypes.c_void_p()
        kc.call("kcStreamCreate", ctypes.byref(s))

        class Buffer(kc.Buffer):
            """A kcMalloc allocation freed with the last state, view or tensor that holds it."""

            def __del__(self):
                self.free()

        class View:
            """A kcMalloc allocation as torch reads it."""

            def __init__(self, buf, shape, dtype):
                self.buf = buf
                kind = {torch.float32: "<f4", torch.float16: "<f2", torch.int32: "<i4", torch.uint8: "|u1", torch.int64: "<i8"}
                self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": kind[dtype], "data": (buf.ptr, False),
                                                 "version": 2}

        _LIB.update(kc=kc, stream=s, Buffer=Buffer, View=View)
    return _LIB


def _empty(*shape, dtype=torch.float32):
    L = _lib()
    b = L["Buffer"](max(1, math.prod(shape)) * torch.empty((), dtype=dtype).element_size())
    return torch.as_tensor(L["View"](b, shape, dtype), device="cuda")


def _own_state(s):
    """The inputs in the library's memory, the outputs and the workspaces: what a program keeps; and the launches."""
    kc, c = _lib()["kc"], s["case"]
    for name, t in list(s.items()):
        if isinstance(t, torch.Tensor):
            s[name] = _empty(*t.shape, dtype=t.dtype)
            s[name].copy_(t)
    at = lambda name: s[name].data_ptr() if name in s else None  # noqa: E731
    if c["kind"] == "store":
        n, row = c["n"], c["n"] // 32 * 18
        s["out"] = _empty(c["rows"], n)
        s["launches"] = [
            ("set_rows_q4_0", kc.SetRowsQ40Args(at("src"), at("idx"), at("cache"), n, c["rows"], n, c["cache"], row)),
            ("get_rows_q4_0", kc.GetRowsQ40Args(at("cache"), at("idx"), at("out"), n, c["rows"], c["cache"], row))]
    elif c["kind"] == "evict":
        K, D, T, n = c["heads_kv"], c["dim"], c["ctx"], c["keep"]
        s["out"] = [_empty(K, n, dtype=torch.int32), _empty(n, K, D, dtype=torch.float16), _empty(n, K, D, dtype=torch.float16),
                    _empty(K, n), _empty(K, n, dtype=torch.int32)]
        keep, k, v, w, pos = (t.data_ptr() for t in s["out"])
        planes = (kc.KvPlane * 4)(kc.KvPlane(at("k"), k, 2 * K * D, 2 * D, 2 * K * D, 2 * D, 2 * D),
                                  kc.KvPlane(at("v"), v, 2 * K * D, 2 * D, 2 * K * D, 2 * D, 2 * D),
                                  kc.KvPlane(at("w"), w, 4, 4 * T, 4, 4 * n, 4),
                                  kc.KvPlane(at("kpos"), pos, 4, 4 * T, 4, 4 * n, 4))
        s["launches"] = [("kv_keep", kc.KvKeepArgs(at("w"), keep, K, T, T, n, n, c["first"], c["recent"])),
                         ("kv_gather", kc.KvGatherArgs(planes, 4, keep, K, n, n, T))]
    else:
        H, K, D, N, T = c["heads"], c["heads_kv"], c["dim"], c["tokens"], c["ctx"]
        head = 2 * D if c["cache"] == "f16" else D // 32 * 18
        d = kc.FlashExtDims(H=H, H_kv=K, D=D, N=N, T=T, q_tok=H * D, q_head=D, m_row=(T + 1) // 2, key_row=T if c["kept"] else 0,
                            pos0=int(s["qpos"][0]), causal=int(c["causal"]), prefix=c["prefix"], k_row=K * head, k_head=head,
                            v_row=K * head, v_head=head)
        shape = dict(q=at("q"), k=at("k"), mask=at("mask"), kpos=at("kpos"), qdoc=at("qdoc"), kdoc=at("kdoc"), slopes=at("slopes"),
                     d=d, scale=1.0 / math.sqrt(D), softcap=c["cap"])
        if c["kind"] == "weights":
            s["out"] = _empty(K, T)
            s["launches"] = [("attn_weights_" + c["cache"], kc.AttnWeightsArgs(
                lse=at("lse"), w_in=at("w_in"), w=at("out"), w_row=T, decay=0.9, **shape))]
        else:
            s["out"] = [_empty(N, H, D)] + ([_empty(N, H)] if c["lse"] else [])
            s["part"] = _empty(kc.flash_ext_part_bytes(d), dtype=torch.uint8)
            s["launches"] = [("flash_ext_" + c["cache"], kc.FlashExtArgs(
                v=at("v"), out=s["out"][0].data_ptr(), lse=s["out"][1].data_ptr() if c["lse"] else None, part=at("part"), **shape))]
            s["out"] = tuple(s["out"]) if c["lse"] else s["out"][0]


def _own_launches(s):
    L = _lib()
    for name, args in s["launches"]:
        L["kc"].launch(name, args, L["stream"])
    return s["out"]


_own_store = _own_attend = _own_weights = _own_evict = _own_launches


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def _pairs(c):
    """(query, key) pairs that a pass scores, for each head."""
    N, T = c["tokens"], c["ctx"]
    if c["dense"]:
        return N * T // 2
    if not c["causal"] or c["kept"]:
        return N * T if not c["docs"] else int(np.bincount(_documents(T, c["docs"]))[_documents(T, c["docs"])[T - N:]].sum())
    i, p = np.arange(T - N, T), c["prefix"]
    last = np.maximum(i + 1, min(p, T))
    if not c["docs"]:
        return int(last.sum())
    ids = _documents(T, c["docs"])
    starts = np.searchsorted(ids, ids[T - N:], side="left")
    ends = np.searchsorted(ids, ids[T - N:], side="right")
    return int(np.maximum(0, np.minimum(last, ends) - starts).sum())


def work(case):
    c = case
    if c["kind"] == "store":
        return {"bytes": c["rows"] * (4 * c["n"] * 2 + 2 * (c["n"] // 32 * 18) + 8), "flops": 2 * c["rows"] * c["n"]}
    if c["kind"] == "evict":
        K, n = c["heads_kv"], c["keep"]
        return {"bytes": K * (4 * c["ctx"] + 4 * n + 2 * n * (4 * c["dim"] + 8)), "flops": 0}
    H, K, D, N, T = c["heads"], c["heads_kv"], c["dim"], c["tokens"], c["ctx"]
    head = 2 * D if c["cache"] == "f16" else D // 32 * 18
    extra = (2 * N * T if c["dense"] else 0) + (4 * K * T if c["kept"] else 0) + (4 * (N + T) if c["docs"] else 0)
    if c["kind"] == "weights":
        return {"bytes": 4 * N * H * (D + 1) + T * K * (head + 8) + extra, "flops": 2 * D * H * _pairs(c)}
    return {"bytes": 8 * N * H * D + 2 * T * K * head + extra, "flops": 4 * D * H * _pairs(c)}
