"""The operators of a serving step for many requests at once, as measurable cases: pages, slots and draft trees of a paged cache from
the requests' lengths, rotary positions with the store into that cache, attention of drafted trees over it, and sampling.

Head counts, widths and vocabularies are the repository's own (32 or 24 query heads of 128 over 8 KV heads, 128256 or 151936
tokens) or generic. Queries, keys and values are N(0, 1), as after their norms. The requests' lengths follow from the case,
everything else from the seed.

`run` gives each operator's plain form in elementary torch operations where `own` is false, and the library's kernels where it
is true."""
import math

import numpy as np
import torch

own = False


# ---- the cases --------------------------------------------------------------------------------------------------

def listed():
    return [
        # eight requests that decode a token each: latency alone
        dict(name="pages_token", kind="pages", seqs=8, ctx=2000, add=1, page=16, tree=False),
        # prompts' chunks and decoding requests of a busy server
        dict(name="pages_chunks", kind="pages", seqs=256, ctx=4001, add=97, page=64, tree=False),
        # drafted trees of every request
        dict(name="pages_trees", kind="pages", seqs=500, ctx=3001, add=24, page=32, tree=True),
        # the query and key heads of eight decoding requests at far positions of a stretched context, keys and values stored
        dict(name="rope_token", kind="rope", tokens=8, heads=32, heads_kv=8, dim=128, n_rot=128, interleaved=False, base=1e6, factor=4.0,
             orig=32768, yarn=True, ctx=120000),
        # a ragged prompt, half of each head rotated in neighbouring pairs
        dict(name="rope_prompt_3333", kind="rope", tokens=3333, heads=24, heads_kv=8, dim=128, n_rot=64, interleaved=True, base=5e5, factor=1.0,
             orig=8192, yarn=False, ctx=3400),
        # one request, one token
        dict(name="tree_token_8k", kind="tree", seqs=1, nodes=1, ctx=8191, heads=32, heads_kv=8, dim=128, page=16, tree=False),
        # one request's drafted tree
        dict(name="tree_24", kind="tree", seqs=1, nodes=24, ctx=2050, heads=24, heads_kv=8, dim=128, page=64, tree=True),
        # a batch of decoding requests of uneven lengths
        dict(name="tokens_128x4k", kind="tree", seqs=128, nodes=1, ctx=4000, heads=32, heads_kv=8, dim=128, page=16, tree=False),
        # a batch of drafted trees
        dict(name="trees_32x4k", kind="tree", seqs=32, nodes=16, ctx=4000, heads=32, heads_kv=8, dim=128, page=32, tree=True),
        # the widest tree over a long context
        dict(name="tree_64_100k", kind="tree", seqs=1, nodes=64, ctx=100003, heads=32, heads_kv=8, dim=128, page=256, tree=True),
        # one decoded token, the usual cuts
        dict(name="sample_row", kind="sample", rows=1, vocab=128256, spread=2.5, top_k=40, top_p=0.95, min_p=0.05),
        # every node of a batch's trees, from the nucleus alone
        dict(name="sample_512_nucleus", kind="sample", rows=512, vocab=151936, spread=2.0, top_k=0, top_p=0.9, min_p=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["pages", "rope", "tree", "tree", "tree", "sample", "sample"])
    if kind == "pages":
        tree = rng.random() < 0.5
        add = _log(rng, 1, 64 if tree else 512)
        return dict(kind=kind, seqs=_log(rng, 1, min(1000, 24000 // add)), ctx=_log(rng, 1, 8000), add=add, page=rng.choice([16, 32, 64, 256]), tree=tree)
    if kind == "rope":
        dim = rng.choice([64, 128, 128, 256])
        heads, heads_kv = rng.choice([(32, 8), (24, 8), (8, 8), (16, 1), (10, 2)])
        stretched = rng.random() < 0.5
        return dict(kind=kind, tokens=_log(rng, 1, 3000 * 128 // dim), heads=heads, heads_kv=heads_kv, dim=dim, n_rot=rng.choice([dim, dim, dim // 2, 32, 10]),
                    interleaved=rng.random() < 0.5, base=rng.choice([1e4, 5e5, 1e6]), factor=rng.choice([2.0, 4.0, 32.0]) if stretched else 1.0,
                    orig=rng.choice([4096, 8192, 32768]), yarn=stretched and rng.random() < 0.7, ctx=_log(rng, 3000, 1000000))
    if kind == "sample":
        return dict(kind=kind, rows=_log(rng, 1, 400), vocab=rng.choice([128256, 151936, _log(rng, 1000, 152000)]), spread=rng.choice([1.0, 2.0, 3.0, 5.0]),
                    top_k=rng.choice([0, 0, 20, 50, _log(rng, 2, 2000)]), top_p=rng.choice([1.0, 0.95, 0.8, 0.5]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]))
    heads, heads_kv = rng.choice([(32, 8), (32, 8), (24, 8), (8, 8), (16, 1), (10, 2)])
    dim = rng.choice([64, 128, 128, 256])
    nodes = rng.choice([1, rng.randint(2, 8), rng.randint(9, 64), rng.randint(9, 64)])
    # (positions of all requests: as many products as the largest listed case has, at most 300000)
    room = min(300000, 100000 * 64 * 32 * 128 // (nodes * heads * dim))
    seqs = _log(rng, 1, min(160, room // 100))
    return dict(kind=kind, seqs=seqs, nodes=nodes, ctx=_log(rng, 80, max(100, min(100000, room // seqs))), heads=heads, heads_kv=heads_kv, dim=dim,
                page=rng.choice([16, 16, 32, 64, 128, 256]), tree=nodes > 1 and rng.random() < 0.7)


# ---- inputs -----------------------------------------------------------------------------------------------------

def _gen(seed, *ids):
    for i in ids:
        seed = (seed * 1000003 + i + 7) & 0x7FFFFFFFFFFF
    return torch.Generator(device="cuda").manual_seed(seed & 0x7FFFFFFFFFFF)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _counts(case, mean, salt):
    """Uneven counts of a case's requests, from about a quarter of their mean to seven quarters; one request has the mean."""
    s = case["seqs"]
    if s == 1 or mean == 1:
        return np.full(s, mean, np.int64)
    f = np.mod((np.arange(s) + salt) * 0.6180339887498949, 1.0)
    return np.maximum(1, np.rint(mean * (0.25 + 1.5 * f))).astype(np.int64)


def _nodes(case):
    return np.minimum(_counts(case, case["nodes"], 3), 64)


def _added(case):
    add = _counts(case, case["add"], 3)
    return np.minimum(add, 64) if case["tree"] else add


def _ints(x, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype).cuda()


def _freqs(c):
    """A pair's revolutions per position, in 64 bits, and the factor on cosine and sine: theta_i = base^(-2 i / n_rot), slowed down
    by `factor`; with yarn, pairs that turn often within the original context keep their speed and those between are blended."""
    n, i = c["n_rot"], np.arange(c["n_rot"] // 2)
    theta = c["base"] ** (-2.0 * i / n)
    if not c["yarn"]:
        return theta / c["factor"] / (2 * math.pi), 1.0
    turns = [n * math.log(c["orig"] / (beta * 2 * math.pi)) / (2 * math.log(c["base"])) for beta in (32.0, 1.0)]
    low, high = max(0, math.floor(turns[0])), min(n - 1, math.ceil(turns[1]))
    slow = np.clip((i - low) / max(0.001, high - low), 0, 1)
    return (theta / c["factor"] * slow + theta * (1 - slow)) / (2 * math.pi), 1 + 0.1 * math.log(c["factor"])


def _closure(parent, start, seqs, nmax):
    """Whether node j of a sequence is node i or one of its ancestors: [seqs, nmax, nmax]."""
    n = parent.shape[0]
    t = torch.arange(n, device=parent.device)
    seq = torch.searchsorted(start[1:].contiguous(), t, right=True)
    a = torch.zeros(seqs, nmax, nmax + 1, device=parent.device)
    a[seq, t - start[seq], parent.long() % (nmax + 1)] = 1.0  # (no parent: the column that is cut off)
    step = a[:, :, :nmax] + torch.eye(nmax, device=parent.device)
    return torch.linalg.matrix_power(step, 64) > 0, seq  # (trees of at most 64 nodes)


def _words(seen, seq, node):
    """Rows of a closure as 64 bits in two int32 words."""
    bits = torch.nn.functional.pad(seen[seq, node], (0, 64 - seen.shape[-1])).view(-1, 2, 32).long()
    return (bits << torch.arange(32, device=bits.device)).sum(-1).int()


def _parents(g, counts, start):
    """A node's parent, by its number in its request's tree: any node before it; the first has none."""
    n = int(counts.sum())
    node = torch.arange(n, device="cuda") - start[:-1].repeat_interleave(_ints(counts, torch.int64), output_size=n)
    return torch.where(node == 0, -1, (torch.rand(n, generator=g, device="cuda") * node).long()).int()


def prepare(case, seed):
    c = dict(case)
    if c["kind"] == "pages":
        have, add = _counts(c, c["ctx"], 0), _added(c)
        P, n = c["page"], int(add.sum())
        held, total = -(-have // P), -(-(have + add) // P)
        width = int(total.max())
        order = torch.randperm(int(total.sum()) + 50, generator=_gen(seed, 1), device="cuda").int()
        table = torch.full((c["seqs"], width), -1, dtype=torch.int32, device="cuda")
        table[_ints(np.repeat(np.arange(c["seqs"]), held), torch.int64),
              _ints(np.concatenate([np.arange(h) for h in held]), torch.int64)] = order[:int(held.sum())]
        t = dict(have=_ints(have), add=_ints(add), table=table, free=order[int(held.sum()):].contiguous())
        if c["tree"]:
            t["parent"] = _parents(_gen(seed, 2), add, _ints(np.concatenate([[0], np.cumsum(add)]), torch.int64))
        s = dict(case=c, n=n, pages=int((total - held).sum()), nmax=int(add.max()), **t)
    elif c["kind"] == "rope":
        N, H, K, D = c["tokens"], c["heads"], c["heads_kv"], c["dim"]
        rows = -(-(N + 1000) // 16) * 16
        turns, scale = _freqs(c)
        s = dict(case=c, q=_normal(_gen(seed, 1), N, H, D), k=_normal(_gen(seed, 2), N, K, D), v=_normal(_gen(seed, 3), N, K, D),
                 slots=torch.randperm(rows, generator=_gen(seed, 4), device="cuda")[:N].contiguous(),
                 pos=torch.randint(max(0, c["ctx"] - N - 100), c["ctx"], (N,), generator=_gen(seed, 5), device="cuda").int(),
                 k_cache=torch.zeros(rows, K, D, dtype=torch.float16, device="cuda"),
                 v_cache=torch.zeros(rows, K, D, dtype=torch.float16, device="cuda"),
                 freqs=torch.from_numpy(turns).cuda(), scale=scale)
    elif c["kind"] == "sample":
        R, V = c["rows"], c["vocab"]
        x = _normal(_gen(seed, 1), R, V) * c["spread"]
        s = dict(case=c, logits=x, u=torch.rand(R, generator=_gen(seed, 2), device="cuda"),
                 temperature=0.5 + torch.rand(R, generator=_gen(seed, 3), device="cuda"),
                 top_k=torch.full((R,), c["top_k"], dtype=torch.int32, device="cuda"),
                 top_p=torch.full((R,), c["top_p"], device="cuda"), min_p=torch.full((R,), c["min_p"], device="cuda"))
    else:
        H, K, D, P = c["heads"], c["heads_kv"], c["dim"], c["page"]
        n, ctx = _nodes(c), _counts(c, c["ctx"], 0)
        length = ctx + n  # (the new tokens' keys and values are in the cache)
        N, held = int(n.sum()), -(-length // P)
        pages = int(held.sum()) + 7
        order = torch.randperm(pages, generator=_gen(seed, 1), device="cuda").int()
        table = torch.full((c["seqs"], int(held.max())), -1, dtype=torch.int32, device="cuda")
        table[_ints(np.repeat(np.arange(c["seqs"]), held), torch.int64),
              _ints(np.concatenate([np.arange(h) for h in held]), torch.int64)] = order[:int(held.sum())]
        start = _ints(np.concatenate([[0], np.cumsum(n)]))
        s = dict(case=c, q=_normal(_gen(seed, 2), N, H, D), table=table, start=start, length=_ints(length), nmax=int(n.max()),
                 lmax=int(length.max()), pages=pages)
        for x, i in (("k", 3), ("v", 4)):
            s[x] = torch.empty(pages * P, K, D, dtype=torch.float16, device="cuda")
            g = _gen(seed, i)
            for r in range(0, pages * P, 1 << 16):
                s[x][r:r + (1 << 16)] = torch.randn(min(1 << 16, pages * P - r), K, D, generator=g, device="cuda").half()
        if c["tree"]:
            parent = _parents(_gen(seed, 5), n, start.long())
            seen, seq = _closure(parent, start.long(), c["seqs"], s["nmax"])
            s["tree"] = _words(seen, seq, torch.arange(N, device="cuda") - start.long()[seq])
    if own:
        _own_state(s)
    torch.cuda.synchronize()
    return s


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


# ---- the plain forms --------------------------------------------------------------------------------------------

def _plain_pages(s):
    c, P, n = s["case"], s["case"]["page"], s["n"]
    have, add, dev = s["have"].long(), s["add"].long(), s["have"].device
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    start = torch.cat([zero, add.cumsum(0)])
    every = torch.arange(c["seqs"], device=dev)
    held = (have + P - 1) // P
    need = (have + add + P - 1) // P - held
    before = torch.cat([zero, need.cumsum(0)])
    to = every.repeat_interleave(need, output_size=s["pages"])
    k = torch.arange(s["pages"], device=dev)
    s["table"][to, held[to] + k - before[to]] = s["free"][:s["pages"]]
    seq = every.repeat_interleave(add, output_size=n)
    node = torch.arange(n, device=dev) - start[seq]
    p = have[seq] + node
    slots = s["table"][seq, p // P].long() * P + p % P
    out = dict(start=start.int(), length=(have + add).int(), slots=slots, used=before[-1:].int(), table=s["table"])
    if not c["tree"]:
        return dict(out, pos=p.int())
    seen, _ = _closure(s["parent"], start, c["seqs"], s["nmax"])
    return dict(out, pos=(have[seq] + seen[seq, node].sum(-1) - 1).int(), tree=_words(seen, seq, node))


def _turn(x, cos, sin, c):
    """The first n_rot values of each head turned: neighbours, or the halves' values of the same number."""
    n = c["n_rot"]
    r = x[..., :n]
    a, b = (r[..., 0::2], r[..., 1::2]) if c["interleaved"] else (r[..., :n // 2], r[..., n // 2:])
    y = a * cos - b * sin, a * sin + b * cos
    y = torch.stack(y, -1).flatten(-2) if c["interleaved"] else torch.cat(y, -1)
    return torch.cat([y, x[..., n:]], -1)


def _plain_rope(s):
    c = s["case"]
    turns = s["pos"].double()[:, None] * s["freqs"]  # (in 64 bits: angles of far positions)
    angle = (turns - turns.floor()) * (2 * math.pi)
    cos, sin = (torch.cos(angle) * s["scale"]).float()[:, None], (torch.sin(angle) * s["scale"]).float()[:, None]
    s["k_cache"][s["slots"]] = _turn(s["k"], cos, sin, c).half()
    s["v_cache"][s["slots"]] = s["v"].half()
    return _turn(s["q"], cos, sin, c), s["k_cache"], s["v_cache"]


def _padded(s):
    """The requests side by side: the tokens of each [seqs, nmax], whether they are there, and the slots of their positions
    [seqs, lmax]."""
    c, P = s["case"], s["case"]["page"]
    start, length = s["start"].long(), s["length"].long()
    i = torch.arange(s["nmax"], device=start.device)
    j = torch.arange(s["lmax"], device=start.device)
    n = start[1:] - start[:-1]
    token = (start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    page = s["table"].long().gather(1, (torch.minimum(j, length[:, None] - 1) // P))
    base = (length - n)[:, None, None]
    node = j[None, None] - base
    if c["tree"]:
        words = s["tree"][token].long()  # (seqs, nmax, 2)
        bit = words.gather(2, (node.clamp(0, 63) // 32).expand(-1, s["nmax"], -1)) >> (node.clamp(0, 63) % 32) & 1
        seen = (node < 0) | ((bit == 1) & (node < n[:, None, None]))
    else:
        seen = node <= i[None, :, None]
    return token, i < n[:, None], page * P + j % P, seen


def _plain_tree(s):
    c = s["case"]
    S, H, K, D, M = c["seqs"], c["heads"], c["heads_kv"], c["dim"], s["nmax"]
    token, there, slot, seen = _padded(s)
    k, v = s["k"][slot].float().transpose(1, 2).contiguous(), s["v"][slot].float().transpose(1, 2).contiguous()
    q = s["q"][token].view(S, M, K, H // K, D).permute(0, 2, 3, 1, 4).reshape(S, K, -1, D)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).view(S, K, H // K, M, -1) * (1.0 / math.sqrt(D))
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    total = x.sum(-1).view(S, K, -1, 1)
    o = torch.matmul(x.view(S, K, -1, s["lmax"]), v) / total
    o = o.view(S, K, H // K, M, D).permute(0, 3, 1, 2, 4).reshape(S * M, H, D)
    # a token's row among the padded ones
    at = torch.arange(s["q"].shape[0], device=token.device)
    seq = torch.searchsorted(s["start"][1:].contiguous(), at.int(), right=True)
    return o[seq * M + at - s["start"].long()[seq]]


def _plain_sample(s):
    # (in 64 bits: which token a number next to a border of the cumulated weights gives)
    R, V = s["logits"].shape
    x, index = torch.sort(s["logits"].double() / s["temperature"].double()[:, None], dim=1, descending=True, stable=True)
    w = torch.exp(x - x[:, :1])
    rank = torch.arange(V, device=x.device)
    k = torch.where(s["top_k"] > 0, s["top_k"].long(), V)[:, None]
    w = torch.where(rank < k, w, 0.0)
    total = w.cumsum(1)
    p = s["top_p"].double()[:, None]
    keep = (rank < k) & ((total - w < p * total[:, -1:]) | (p >= 1)) & (w >= s["min_p"].double()[:, None]) | (rank == 0)
    last = keep.sum(1, keepdim=True) - 1
    whole = total.gather(1, last)
    at = (total <= s["u"].double()[:, None] * whole).sum(1, keepdim=True).minimum(last)
    return index.gather(1, at)[:, 0].int(), (w.gather(1, at) / whole)[:, 0].float()


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------

def exact(case, seed):
    c = dict(case)
    if c["kind"] == "pages":
        return None  # (whole numbers)
    t = prepare(case, seed)
    if c["kind"] == "rope":
        turns, scale = _freqs(c)
        n = c["n_rot"]
        z = torch.polar(torch.ones(c["tokens"], n // 2, dtype=torch.float64, device="cuda"),
                        torch.remainder(t["pos"].double()[:, None] * torch.from_numpy(turns).cuda(), 1.0) * (2 * math.pi))[:, None] * scale

        def turned(x):
            y = x.double().clone()
            i = torch.arange(n // 2, device="cuda")
            a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + n // 2)
            w = torch.complex(y[..., a], y[..., b]) * z
            y[..., a], y[..., b] = w.real, w.imag
            return y
        kc, vc = torch.zeros_like(t["k_cache"], dtype=torch.float64), torch.zeros_like(t["v_cache"], dtype=torch.float64)
        kc[t["slots"]], vc[t["slots"]] = turned(t["k"]), t["v"].double()
        return turned(t["q"]), kc, vc
    if c["kind"] == "sample":
        probs = []
        for r in range(c["rows"]):  # from the definition: ranks, then cuts of the ranked list
            z = t["logits"][r].double() / t["temperature"][r].double()
            order = torch.argsort(-z, stable=True)
            w = torch.exp(z[order] - z[order[0]])
            if c["top_k"]:
                w = w[:c["top_k"]]
            cut = int((w >= t["min_p"][r].double()).sum())
            if c["top_p"] < 1:
                cut = min(cut, int((torch.cumsum(w, 0) < t["top_p"][r].double() * w.sum()).sum()) + 1)
            w = w[:max(1, cut)] / w[:max(1, cut)].sum()
            probs.append(w[min(len(w) - 1, int((torch.cumsum(w, 0) <= t["u"][r].double()).sum()))])
        return None, torch.stack(probs)
    K, D, P, G = c["heads_kv"], c["dim"], c["page"], c["heads"] // c["heads_kv"]
    start, length = t["start"].tolist(), t["length"].tolist()
    out = torch.empty(t["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(c["seqs"]):
        a, b, n = start[i], length[i], start[i + 1] - start[i]
        slots = (t["table"][i, :-(-b // P)].long()[:, None] * P + torch.arange(P, device="cuda")).flatten()[:b]
        seen = torch.ones(n, b, dtype=torch.bool, device="cuda")
        if c["tree"]:
            w = t["tree"][a:a + n].cpu().numpy().view(np.uint32).astype(np.uint64)
            w = w[:, 0] | w[:, 1] << np.uint64(32)
            seen[:, b - n:] = torch.from_numpy((w[:, None] >> np.arange(n, dtype=np.uint64) & np.uint64(1)).astype(bool)).cuda()
        else:
            seen[:, b - n:] = torch.ones(n, n, device="cuda").tril() > 0
        for g in range(K):
            keys, values = t["k"][slots, g].double(), t["v"][slots, g].double()
            x = t["q"][a:a + n, g * G:(g + 1) * G].double() @ keys.t() / math.sqrt(D)
            x = torch.where(seen[:, None], x, -math.inf)
            out[a:a + n, g * G:(g + 1) * G] = torch.softmax(x, -1) @ values
    return out


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
                kind = {torch.float32: "<f4", torch.float16: "<f2", torch.float64: "<f8", torch.int32: "<i4", torch.uint8: "|u1", torch.int64: "<i8"}
                self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": kind[dtype], "data": (buf.ptr, False),
                                                 "version": 2}

        _LIB.update(kc=kc, stream=s, Buffer=Buffer, View=View)
    return _LIB


def _empty(*shape, dtype=torch.float32):
    L = _lib()
    b = L["Buffer"](max(1, math.prod(shape)) * torch.empty((), dtype=dtype).element_size())
    return torch.as_tensor(L["View"](b, shape, dtype), device="cuda")


def _own_state(s):
    """The inputs in the library's memory, the outputs and the workspaces: what a program keeps; and the launch."""
    kc, c = _lib()["kc"], s["case"]
    for name, t in list(s.items()):
        if isinstance(t, torch.Tensor):
            s[name] = _empty(*t.shape, dtype=t.dtype)
            s[name].copy_(t)
    at = lambda name: s[name].data_ptr() if name in s else None  # noqa: E731
    if c["kind"] == "pages":
        n, S, i32 = s["n"], c["seqs"], torch.int32
        o = dict(start=_empty(S + 1, dtype=i32), length=_empty(S, dtype=i32), slots=_empty(n, dtype=torch.int64), used=_empty(1, dtype=i32),
                 table=s["table"], pos=_empty(n, dtype=i32))
        if c["tree"]:
            o["tree"] = _empty(n, 2, dtype=i32)
        p = {k: v.data_ptr() for k, v in o.items()}
        s["launch"] = "kv_pages", kc.KvPagesArgs(
            have=at("have"), add=at("add"), free=at("free"), parent=at("parent"), table=p["table"], start=p["start"], len=p["length"], slots=p["slots"],
            pos=p["pos"], used=p["used"], tree=p.get("tree"), seqs=S, n_tokens=n, n_free=s["free"].shape[0], page=c["page"],
            max_pages=s["table"].shape[1], table_row=s["table"].shape[1], tree_words=2 if c["tree"] else 0)
    elif c["kind"] == "rope":
        N, H, K, D = c["tokens"], c["heads"], c["heads_kv"], c["dim"]
        o = _empty(N, H, D), s["k_cache"], s["v_cache"]
        turns, scale = kc.rope_freqs(c["n_rot"], c["base"], factor=c["factor"], yarn_ctx=c["orig"] if c["yarn"] else 0)
        s["freqs"].copy_(torch.from_numpy(turns))
        s["launch"] = "rope_ext", kc.RopeExtArgs(
            q=at("q"), k=at("k"), v=at("v"), pos=at("pos"), freqs=at("freqs"), slots=at("slots"), q_out=o[0].data_ptr(), k_cache=at("k_cache"),
            v_cache=at("v_cache"), n_tokens=N, H=H, H_kv=K, D=D, n_rot=c["n_rot"], interleaved=int(c["interleaved"]), q_tok=H * D, q_head=D,
            k_tok=K * D, k_head=D, v_tok=K * D, v_head=D, out_tok=H * D, out_head=D, cache_rows=s["k_cache"].shape[0], kc_row=2 * K * D, kc_head=2 * D,
            vc_row=2 * K * D, vc_head=2 * D, scale=scale)
    elif c["kind"] == "sample":
        R, V = c["rows"], c["vocab"]
        o = _empty(R, dtype=torch.int32), _empty(R)
        s["part"] = _empty(kc.sample_rows_part_bytes(R, V), dtype=torch.uint8)
        s["launch"] = "sample_rows", kc.SampleRowsArgs(
            logits=at("logits"), u=at("u"), temperature=at("temperature"), top_k=at("top_k"), top_p=at("top_p"), min_p=at("min_p"),
            tokens=o[0].data_ptr(), probs=o[1].data_ptr(), part=at("part"), row=V, rows=R, n_vocab=V)
    else:
        H, K, D, N = c["heads"], c["heads_kv"], c["dim"], s["q"].shape[0]
        d = kc.FlashPagesDims(H=H, H_kv=K, D=D, N=N, seqs=c["seqs"], page=c["page"], max_pages=s["table"].shape[1], n_pages=s["pages"],
                              tree_words=2 if c["tree"] else 0, q_tok=H * D, q_head=D, table_row=s["table"].shape[1],
                              k_row=2 * K * D, k_head=2 * D, v_row=2 * K * D, v_head=2 * D)
        o = _empty(N, H, D)
        s["part"] = _empty(kc.flash_pages_part_bytes(d), dtype=torch.uint8)
        s["launch"] = "flash_pages_f16", kc.FlashPagesArgs(
            q=at("q"), k=at("k"), v=at("v"), table=at("table"), start=at("start"), len=at("length"), tree=at("tree"), out=o.data_ptr(), part=at("part"),
            d=d, scale=1.0 / math.sqrt(D))
    s["out"] = o


def _own_launch(s):
    L = _lib()
    L["kc"].launch(*s["launch"], L["stream"])
    return s["out"]


_own_pages = _own_rope = _own_tree = _own_sample = _own_launch


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "pages":
        have, add, P = _counts(c, c["ctx"], 0), _added(c), c["page"]
        n, new = int(add.sum()), int((-(-(have + add) // P) - -(-have // P)).sum())
        return {"bytes": 16 * c["seqs"] + (16 + (12 if c["tree"] else 0)) * n + 8 * new, "flops": 4 * n}
    if c["kind"] == "rope":
        H, K, D = c["heads"], c["heads_kv"], c["dim"]
        return {"bytes": c["tokens"] * (8 * H * D + 12 * K * D + 12) + 4 * c["n_rot"], "flops": 3 * c["tokens"] * (H + K) * c["n_rot"]}
    if c["kind"] == "sample":
        return {"bytes": 4 * c["rows"] * c["vocab"] + 28 * c["rows"], "flops": 10 * c["rows"] * c["vocab"]}
    H, K, D = c["heads"], c["heads_kv"], c["dim"]
    n, ctx = _nodes(c), _counts(c, c["ctx"], 0)
    pairs = int((n * ctx).sum() + (n * (n + 1) // 2).sum())  # (a tree's nodes see no more than that of each other)
    return {"bytes": 8 * int(n.sum()) * H * D + 4 * K * D * int((ctx + n).sum()) + 4 * int((-(-(ctx + n) // c["page"])).sum()), "flops": 4 * D * H * pairs}
