"""flash_pages_f16 against its definition in 64 bits (tests/serve.py derives the bounds), at the lengths, trees, pages and layouts where
it can go wrong."""
import ctypes as C

import numpy as np
import pytest

import kernelcore_amd as kc
from tests.serve import Out, Pages, up

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def runtime():
    kc.init()
    yield
    kc.synchronize()


@pytest.fixture(autouse=True, params=[0, 1 << 26], ids=["", "room"])
def room(request, monkeypatch):
    """Tables as long as the sequences, and with room for more work than the form for little of it takes."""
    monkeypatch.setattr(Pages, "room", request.param)


HEADS = [(8, 2, 128), (6, 2, 64), (4, 2, 256), (32, 8, 128), (5, 5, 64), (16, 1, 128), (17, 1, 64), (10, 2, 256), (4, 4, 128)]


@pytest.mark.parametrize("H,K,D", HEADS)
@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("lens", [[1], [31], [32], [33], [64, 1, 129], [127, 500, 16, 17], [1025], [2047, 3]], ids=str)
def test_tokens(H, K, D, page, lens):
    """One token a sequence."""
    print("flash_pages", H, K, D, page, lens, flush=True)
    Pages(H, K, D, lens, [1] * len(lens), page, tree=False).check()


@pytest.mark.parametrize("H,K,D", HEADS)
@pytest.mark.parametrize("tree", [False, True], ids=["causal", "tree"])
@pytest.mark.parametrize("lens,nodes", [([5], [5]), ([300], [17]), ([40, 64, 65], [2, 64, 33]), ([600, 100, 9], [24, 7, 9]), ([513], [64]), ([1500, 200], [50, 41]),
                                        ([700], [300]), ([129, 257], [129, 200])], ids=str)
def test_nodes(H, K, D, tree, lens, nodes):
    print("flash_pages", H, K, D, tree, lens, nodes, flush=True)
    Pages(H, K, D, lens, nodes, 32, tree=tree, words=10 if max(nodes) > 64 else 2).check()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_uneven(D):
    """Sequences of no token, of no position but their own, of none at all, long ones beside short ones."""
    lens = [0, 7, 2000, 33, 0, 900, 1, 64, 5, 3111]
    nodes = [0, 0, 3, 20, 0, 0, 1, 64, 5, 1]
    Pages(8, 2, D, lens, nodes, 16, tree=True).check()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nodes", [1, 3, 40])
def test_no_positions(D, nodes):
    """Fewer positions than tokens (none at all, or some): the first tokens see nothing."""
    for n in (0, 1, nodes - 1):
        c = Pages(4, 2, D, [max(0, n), 50], [nodes, 2], 16, tree=False)
        out, sums = c.check()
        # token i sees the positions up to itself, counted from the end: none where fewer are there
        first = nodes - max(0, n)
        assert (out[:first] == 0).all() and np.isneginf(sums[:first]).all()


@pytest.mark.parametrize("words,nodes", [(1, 40), (1, 32), (3, 96), (3, 200), (64, 300)])
def test_tree_words(words, nodes):
    """Nodes past the words' bits are seen by none, themselves neither."""
    Pages(6, 2, 64, [nodes + 70, nodes], [nodes, nodes], 16, tree=True, words=words).check()


@pytest.mark.parametrize("H,K,D", [(8, 2, 128), (8, 2, 64), (4, 2, 256)])
@pytest.mark.parametrize("seqs,nodes", [(300, 1), (900, 1), (150, 5), (70, 24)])
def test_many_sequences(H, K, D, seqs, nodes):
    print("flash_pages", H, K, D, seqs, nodes, flush=True)
    r = np.random.default_rng(seqs)
    n = np.minimum(r.integers(0, 2 * nodes + 1, seqs), 64)
    Pages(H, K, D, n + r.integers(0, 150, seqs), n, 16, tree=nodes > 1).check()


@pytest.mark.parametrize("H,K,D,nodes", [(8, 2, 128, 1), (32, 8, 128, 16), (4, 1, 64, 64), (8, 2, 256, 9)])
def test_long(H, K, D, nodes):
    """A sequence that is divided among many workgroups, beside others."""
    Pages(H, K, D, [20011, 100, 6007], [nodes, nodes, nodes], 256, tree=True).check()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nodes", [1, 20])
def test_pages_not_there(D, nodes):
    """Positions of pages outside the cache are not seen; a table full of them leaves nothing."""
    c = Pages(8, 2, D, [500, 300, 90], [nodes] * 3, 16, tree=False)
    c.table[0, [0, 3, 17]] = [-1, c.n_pages, 2**31 - 1]
    c.table[1, :] = -5
    out, sums = c.check()
    assert (out[nodes:2 * nodes] == 0).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nodes", [1, 8, 30])
def test_short_table(D, nodes):
    """A length past the table's end: positions end with the table."""
    c = Pages(4, 2, D, [96, 200], [nodes, nodes], 16, tree=False)
    want = c.check()[0]
    b = c.upload()
    d = c.dims(max_pages=6, table_row=c.max_pages)
    part, out = Out(kc.flash_pages_part_bytes(d), np.uint8), Out(c.q.size, np.float32)
    kc.launch("flash_pages_f16", kc.FlashPagesArgs(**{k: x.ptr for k, x in b.items()}, out=out.ptr, part=part.ptr, d=d, scale=c.scale))
    kc.synchronize()
    got = out.get().reshape(c.q.shape)
    part.get()
    assert np.array_equal(got[:nodes], want[:nodes]) or np.allclose(got[:nodes], want[:nodes], atol=1e-5)
    # (the second sequence's 200 positions end with 96: its tokens, from 200 - nodes on, see those alike)
    e = Pages(4, 2, D, [96, 200], [nodes, nodes], 16, tree=False)
    e.lens = np.array([96, 96])
    e.nodes = np.array([nodes, 0])
    slot = e.slots(1)
    for h in range(4):
        x = c.q[nodes:, h].astype(np.float64) @ e.k[slot, h // 2].astype(np.float64).T * c.scale
        p = np.exp(x - x.max(-1, keepdims=True))
        y = p / p.sum(-1, keepdims=True) @ e.v[slot, h // 2].astype(np.float64)
        assert np.abs(got[nodes:, h] - y).max() < 2e-5  # (bounds as in check, for scores below 8)
    for x in b.values():
        x.free()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nodes", [2, 30])
def test_hidden_infinities(D, nodes):
    """What a token does not see (another branch) may hold anything."""
    c = Pages(8, 2, D, [200, 333], [nodes, nodes], 16, tree=True, parent=np.array(([-1] + [0] * (nodes - 1)) * 2))
    hidden = c.slots(0)[-1], c.slots(1)[-1]  # the last node of each: a leaf
    for x in hidden:
        c.k[x], c.v[x] = np.nan, np.nan
    out, sums = c.attend()
    for s in range(2):  # the leaf itself sees its own NaN
        leaf = int(c.start[s + 1]) - 1
        assert np.isnan(out[leaf]).all() and np.isnan(sums[leaf]).all()
    for x in hidden:
        c.k[x], c.v[x] = 0.0, 0.0
    want, bound, lse, lse_bound = c.expected()
    keep = np.ones(c.N, bool)
    keep[[int(x) - 1 for x in c.start[1:]]] = False
    assert (np.abs(out - want) <= bound)[keep].all() and (np.abs(sums - lse) <= lse_bound)[keep].all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nodes", [1, 3, 30])
def test_seen_infinities(D, nodes):
    """A key whose score is -infinity has weight 0; one of +infinity or NaN makes the token NaN; an infinite value comes out so."""
    c = Pages(4, 2, D, [150 + nodes] * 4, [nodes] * 4, 16, tree=False)
    c.q = np.abs(c.q) + np.float32(0.1)
    at = [c.slots(s)[70] for s in range(4)]
    c.k[at[0]] = -np.inf
    c.k[at[1]] = np.inf
    c.k[at[2], :, 0] = np.nan
    c.v[at[3], :, 5] = -np.inf
    out, sums = c.attend()
    n = nodes
    assert np.isnan(out[n:3 * n]).all() and np.isnan(sums[n:3 * n]).all()
    want, bound, lse, lse_bound = c.expected()
    assert (np.abs(out - want) <= bound)[:n].all() and (np.abs(sums - lse) <= lse_bound)[:n].all()
    assert np.isneginf(out[3 * n:, :, 5]).all()
    rest = np.arange(D) != 5
    assert (np.abs(out - want) <= bound)[3 * n:][:, :, rest].all() and (np.abs(sums - lse) <= lse_bound)[3 * n:].all()


def test_scale_and_sizes_of_q():
    for scale, spread in ((0.0, 1.0), (-0.3, 1.0), (1e-30, 1e30), (3.0, 1e-3), (1e20, 1e-20)):
        Pages(8, 2, 128, [300, 77], [1, 9], 16, tree=False, scale=scale, spread=spread).check()


def test_sharp():
    """Scores far apart: the running maximum moves, early sums vanish."""
    for nodes in (1, 30):
        c = Pages(4, 2, 128, [2000], [nodes], 16, tree=False, spread=30.0)
        c.k[c.slots(0)] *= np.linspace(0.1, 2.0, 2000)[:, None, None].astype(np.float16)
        c.check()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("nodes", [1, 20])
def test_strides(D, nodes):
    """q rows and heads apart, K with heads outermost, V rows of another stride, table rows apart; no lse."""
    c = Pages(6, 3, D, [333, 64, 1], [nodes, nodes, 1], 32, tree=False)
    want = c.attend(extra=0)[0]  # (the same sizes: N takes part in how a call is divided)
    qrow, qhead = 6 * (D + 3) + 5, D + 3
    q = np.full(c.N * qrow, np.nan, np.float32)
    np.lib.stride_tricks.as_strided(q, c.q.shape, (4 * qrow, 4 * qhead, 4))[...] = c.q
    rows = c.n_pages * c.page
    khead, vrow, vhead = rows * (2 * D + 16), 3 * (2 * D + 32) + 48, 2 * D + 32
    k, v = np.full(3 * khead // 2, np.nan, np.float16), np.full(rows * vrow // 2, np.nan, np.float16)
    np.lib.stride_tricks.as_strided(k, c.k.shape, (2 * D + 16, khead, 2))[...] = c.k
    np.lib.stride_tricks.as_strided(v, c.v.shape, (vrow, vhead, 2))[...] = c.v
    table = np.full((3, c.max_pages + 9), -1, np.int32)
    table[:, :c.max_pages] = c.table
    b = dict(q=up(q, np.float32), k=up(k, np.float16), v=up(v, np.float16), table=up(table, np.int32), start=up(c.start, np.int32), len=up(c.lens, np.int32))
    d = c.dims(q_tok=qrow, q_head=qhead, k_row=2 * D + 16, k_head=khead, v_row=vrow, v_head=vhead, table_row=c.max_pages + 9)
    part, out = Out(kc.flash_pages_part_bytes(d), np.uint8), Out(c.q.size, np.float32)
    kc.launch("flash_pages_f16", kc.FlashPagesArgs(**{n: x.ptr for n, x in b.items()}, out=out.ptr, part=part.ptr, d=d, scale=c.scale))
    kc.synchronize()
    part.get()
    assert np.array_equal(out.get().reshape(c.q.shape), want)
    for x in b.values():
        x.free()


@pytest.mark.parametrize("nodes", [1, 20])
def test_far_slots(nodes):
    """Rows 1 MiB apart: slots past 4 GiB."""
    c = Pages(2, 1, 64, [70 + nodes, 40 + nodes], [nodes, nodes], 16, tree=False, spare=300)
    row = 1 << 20
    want = c.attend(extra=0)[0]
    far = max(int(c.slots(s).max()) for s in range(2))
    assert far * row > 4 << 30
    kb, vb = kc.Buffer((c.n_pages * 16 - 1) * row + 128), kc.Buffer(c.v.nbytes)
    for s in range(2):
        for x in c.slots(s):
            kb.upload(c.k[x], int(x) * row)
    vb.upload(c.v)
    b = dict(q=up(c.q, np.float32), table=up(c.table, np.int32), start=up(c.start, np.int32), len=up(c.lens, np.int32))
    d = c.dims(k_row=row)
    part, out = Out(kc.flash_pages_part_bytes(d), np.uint8), Out(c.q.size, np.float32)
    kc.launch("flash_pages_f16", kc.FlashPagesArgs(**{n: x.ptr for n, x in b.items()}, k=kb.ptr, v=vb.ptr, out=out.ptr, part=part.ptr, d=d, scale=c.scale))
    kc.synchronize()
    part.get()
    assert np.array_equal(out.get().reshape(c.q.shape), want)
    for x in [kb, vb, *b.values()]:
        x.free()


def test_two_streams():
    """Calls under way together, each with its own workspace."""
    cases = [Pages(8, 2, 128, [3000, 500], [5, 9], 16, seed=i) for i in range(4)]
    want = [c.attend(extra=0)[0] for c in cases]
    made = []
    for c in cases:
        s = C.c_void_p()
        kc.call("kcStreamCreate", C.byref(s))
        b, d = c.upload(), c.dims()
        part, out = kc.Buffer(kc.flash_pages_part_bytes(d)), Out(c.q.size, np.float32)
        made.append((s, kc.FlashPagesArgs(**{n: x.ptr for n, x in b.items()}, out=out.ptr, part=part.ptr, d=d, scale=c.scale), b, part, out))
    for _ in range(5):
        for s, args, *_ in made:
            kc.launch("flash_pages_f16", args, s)
    kc.synchronize()
    for (s, _, b, part, out), w in zip(made, want):
        assert np.array_equal(out.get().reshape(w.shape), w)
        kc.call("kcStreamDestroy", s)
        for x in [part, *b.values()]:
            x.free()


@pytest.mark.parametrize("nodes", [1, 12])
def test_captured(nodes):
    """One captured call serves steps of other lengths, and its results are those of a call on its own."""
    seqs, longest = 5, 700
    r = np.random.default_rng(nodes)
    c = Pages(8, 2, 128, [longest] * seqs, [nodes] * seqs, 16, tree=False)
    b, d = c.upload(), c.dims()
    part, out = kc.Buffer(kc.flash_pages_part_bytes(d)), kc.Buffer(4 * c.q.size)
    s, g = C.c_void_p(), C.c_void_p()
    kc.call("kcStreamCreate", C.byref(s))
    kc.call("kcStreamBeginCapture", s)
    kc.launch("flash_pages_f16", kc.FlashPagesArgs(**{n: x.ptr for n, x in b.items()}, out=out.ptr, part=part.ptr, d=d, scale=c.scale), s)
    kc.call("kcStreamEndCapture", s, C.byref(g))
    for step in range(4):
        c.lens = r.integers(nodes, longest + 1, seqs)
        b["len"].upload(c.lens.astype(np.int32))
        out.upload(np.full(c.q.size, 7.0, np.float32))
        kc.call("kcGraphLaunch", g, s)
        kc.synchronize()
        got = out.download(np.float32).reshape(c.q.shape)
        want, bound, _, _ = c.expected()
        assert (np.abs(got - want) <= bound).all(), step
        kc.launch("flash_pages_f16", kc.FlashPagesArgs(**{n: x.ptr for n, x in b.items()}, out=out.ptr, part=part.ptr, d=d, scale=c.scale), s)
        kc.synchronize()
        assert np.array_equal(out.download(np.float32).reshape(c.q.shape), got), step
    kc.call("kcGraphDestroy", g)
    kc.call("kcStreamDestroy", s)
    for x in [part, out, *b.values()]:
        x.free()
