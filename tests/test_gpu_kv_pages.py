"""kv_pages against its definition, every output bit for bit (tests/serve.py)."""
import numpy as np
import pytest

import kernelcore_amd as kc
from tests.serve import plain_pages, run_pages

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def runtime():
    kc.init()
    yield
    kc.synchronize()


def check(have, add, page, n_tokens=None, n_free=None, max_pages=None, parent=None, words=0, row=None, seed=0, table=None):
    r = np.random.default_rng(seed)
    have, add = np.asarray(have, np.int64), np.asarray(add, np.int64)
    h, a = np.maximum(have, 0), np.maximum(add, 0)
    n_tokens = int(a.sum()) if n_tokens is None else n_tokens
    need = int((-(-(h + a) // page) - -(-h // page)).sum())
    max_pages = max(1, int((-(-(h + a) // page)).max(initial=1))) if max_pages is None else max_pages
    free = r.permutation(need + 5 if n_free is None else n_free).astype(np.int32) + 100000
    if table is None:
        table = r.integers(0, 90000, (len(have), max_pages)).astype(np.int32)
    want = plain_pages(have, add, free, table, page, n_tokens, parent, words)
    got = run_pages(have, add, free, table, page, n_tokens, parent, words, row)
    for k in want:
        assert np.array_equal(got[k], want[k]), (k, np.argwhere(got[k] != want[k])[:4].tolist())


@pytest.mark.parametrize("page", [16, 32, 1024, 65536])
@pytest.mark.parametrize("seqs,most,ctx", [(1, 1, 1), (1, 1, 40), (3, 40, 100), (17, 1, 3000), (64, 300, 500), (257, 9, 77), (1023, 3, 50), (1024, 2, 50),
                                           (1025, 4, 50), (2500, 5, 33)])
def test_ragged(page, seqs, most, ctx):
    print(f"kv_pages page={page} seqs={seqs} add<={most} have<={ctx}", flush=True)
    r = np.random.default_rng([page, seqs, most])
    check(r.integers(0, ctx + 1, seqs), r.integers(0, most + 1, seqs), page, row=5000, seed=seqs)


@pytest.mark.parametrize("have,add,page,kw", [
    ([], [], 16, dict(n_tokens=0)), ([], [], 16, dict(n_tokens=300)), ([0], [0], 16, {}), ([5], [0], 16, dict(n_tokens=3)),
    ([0, 0, 0], [0, 16, 0], 16, {}), ([15, 16, 17], [1, 1, 1], 16, {}), ([16] * 5, [16] * 5, 16, {}),
    ([-5, 3, -1], [4, -7, 2], 16, {}), ([10, 20], [300, 300], 32, dict(n_tokens=450)), ([10, 20, 5], [300, 300, 9], 32, dict(n_tokens=310)),
    ([10, 20, 5], [300, 300, 9], 32, dict(n_tokens=310, n_free=3)), ([0, 0], [100, 100], 16, dict(n_free=0)), ([0, 0], [100, 100], 16, dict(n_free=7)),
    ([30, 90], [60, 60], 16, dict(max_pages=3)), ([1000, 0], [20, 20], 16, dict(max_pages=2)), ([7], [5], 16, dict(n_tokens=600, max_pages=0, table=np.zeros((1, 0), np.int32))),
    ([2**31 - 30], [20], 65536, dict(max_pages=3)), ([2**31 - 1], [2**31 - 1], 16, dict(n_tokens=20, max_pages=3, n_free=2)),
    ([0] * 700, [2**31 - 1] * 700, 16, dict(n_tokens=1000, max_pages=4, n_free=9)), ([3], [5000], 16, {}), ([0] * 3000 + [7], [0] * 3000 + [513], 16, {}),
], ids=str)
def test_edges(have, add, page, kw):
    print("kv_pages", len(have), page, kw.keys(), flush=True)
    check(have, add, page, **kw)


def test_pages_not_there():
    """A negative entry of the table is no page; its positions have no slot."""
    table = np.array([[-1, 5, 7], [3, -9, 1]], np.int32)
    check([10, 20], [30, 20], 16, table=table)


@pytest.mark.parametrize("words", [1, 2, 3, 64])
@pytest.mark.parametrize("kind", ["random", "chain", "flat", "wild"])
@pytest.mark.parametrize("nodes", [[1], [7, 0, 64, 33], [24] * 40, [300, 5, 700, 1]])
def test_trees(words, kind, nodes):
    r = np.random.default_rng([words, len(nodes)])
    parent = []
    for n in nodes:
        i = np.arange(n)
        parent.append(dict(random=np.where(i == 0, -1, (r.random(n) * i).astype(int)), chain=i - 1, flat=np.where(i == 0, -1, 0),
                           wild=r.choice([-5, -1, 0, 1, 2, n - 1, n, 10**6], n))[kind])
    check(r.integers(0, 100, len(nodes)), nodes, 16, parent=np.concatenate(parent), words=words)


def test_repeated_and_captured():
    """A captured call is launched again over other counts, as a serving loop does; padding behind the last token is marked."""
    import ctypes as C
    seqs, n_tokens, page, max_pages, n_free = 6, 64, 16, 8, 200
    r = np.random.default_rng(3)
    table = np.full((seqs, max_pages), -1, np.int32)
    b = {k: kc.Buffer(4 * n) for k, n in dict(have=seqs, add=seqs, free=n_free, table=seqs * max_pages, start=seqs + 1, len=seqs, pos=n_tokens, used=1,
                                              parent=n_tokens, tree=2 * n_tokens).items()}
    b["slots"] = kc.Buffer(8 * n_tokens)
    s = C.c_void_p()
    kc.call("kcStreamCreate", C.byref(s))
    args = kc.KvPagesArgs(**{k: x.ptr for k, x in b.items()}, seqs=seqs, n_tokens=n_tokens, n_free=n_free, page=page, max_pages=max_pages,
                          table_row=max_pages, tree_words=2)
    kc.call("kcStreamBeginCapture", s)
    kc.launch("kv_pages", args, s)
    g = C.c_void_p()
    kc.call("kcStreamEndCapture", s, C.byref(g))
    have = np.zeros(seqs, np.int32)
    b["table"].upload(table)
    for step in range(5):
        add = r.integers(0, 11, seqs).astype(np.int32)
        free = r.permutation(n_free).astype(np.int32)
        parent = (r.random(n_tokens) * 12).astype(np.int32) - 1
        for k, x in dict(have=have, add=add, free=free, parent=parent).items():
            b[k].upload(x)
        want = plain_pages(have, add, free, table, page, n_tokens, parent, 2)
        kc.call("kcGraphLaunch", g, s)
        kc.synchronize()
        for k, x in want.items():
            assert np.array_equal(b[k].download(x.dtype).reshape(x.shape), x), (step, k)
        table, have = want["table"], want["len"]
    kc.call("kcGraphDestroy", g)
    kc.call("kcStreamDestroy", s)
    for x in b.values():
        x.free()
