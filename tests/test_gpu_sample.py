"""sample_rows against its definition in 64 bits (tests/serve.py)."""
import ctypes as C

import numpy as np
import pytest

import kernelcore_amd as kc
from tests.serve import Out, plain_sample, run_sample, up

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def runtime():
    kc.init()
    yield
    kc.synchronize()


def check(l, u, temperature=None, top_k=None, top_p=None, min_p=None, **kw):
    R = len(l)
    at = lambda x, r, d: d if x is None else np.broadcast_to(x, R)[r].item()  # noqa: E731
    tokens, probs = run_sample(l, u, temperature, top_k, top_p, min_p, **kw)
    for r in range(R):
        want, pr = plain_sample(l[r], u[r], at(temperature, r, 1.0), at(top_k, r, 0), at(top_p, r, 1.0), at(min_p, r, 0.0))
        assert tokens[r] in want, (r, tokens[r], want, u[r])
        p = pr[want.index(tokens[r])]
        # (two roundings to 32 bits, steps of 2^-43 of the largest weight)
        assert abs(probs[r] - p) <= 2.0 ** -23 * p + 2.0 ** -40, (r, probs[r], p)
    return tokens


SIZES = [1, 2, 63, 64, 65, 1000, 4097, 16383, 16384, 16385, 32769, 128256, 151936]


@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("spread", [0.0, 0.3, 2.5, 30.0])
def test_cuts(V, spread):
    """Every combination of the cuts, a row each."""
    print("sample_rows", V, spread, flush=True)
    r = np.random.default_rng([V, int(10 * spread)])
    combos = [(t, k, p, m) for t in (1.0, 0.6) for k in (0, 1, 7, 500) for p in (1.0, 0.95, 0.3) for m in (0.0, 0.1)]
    if V > 20000:
        combos = combos[::5] + combos[1::7]
    t, k, p, m = (np.array(x) for x in zip(*combos))
    l = (r.standard_normal((len(combos), V)) * spread).astype(np.float32)
    check(l, r.random(len(combos)).astype(np.float32), t.astype(np.float32), k.astype(np.int32), p.astype(np.float32), m.astype(np.float32))


@pytest.mark.parametrize("V,rows", [(1000, 700), (50000, 130), (151936, 110)])
def test_many_rows(V, rows):
    """Pieces of either size."""
    print("sample_rows", V, rows, flush=True)
    r = np.random.default_rng(V)
    l = (r.standard_normal((rows, V)) * 2).astype(np.float32)
    tokens, probs = run_sample(l, r.random(rows).astype(np.float32), top_p=0.9)
    few = r.permutation(rows)[:12]
    u = np.random.default_rng(V)
    u.standard_normal((rows, V))
    us = u.random(rows).astype(np.float32)
    for i in few:
        want, pr = plain_sample(l[i], us[i], top_p=0.9)
        assert tokens[i] in want and abs(probs[i] - pr[want.index(tokens[i])]) < 1e-6


@pytest.mark.parametrize("V", [65536, 65537, 1 << 20])
@pytest.mark.parametrize("rows", [1, 2, 9])
@pytest.mark.parametrize("kw", [dict(top_k=40), dict(top_p=0.8), {}], ids=str)
def test_large_vocabulary(V, rows, kw):
    """Few rows in small pieces and in large ones; borders among the first tokens, and where most logits are read again."""
    print("sample_rows", V, rows, kw, flush=True)
    r = np.random.default_rng([V, rows])
    l = (r.standard_normal((rows, V)) * 1.5).astype(np.float32)
    check(l, r.random(rows).astype(np.float32), **kw)


@pytest.mark.parametrize("V", [1, 100, 5000, 40000, 128256])
def test_ties(V):
    """Equal logits are ordered by their number, also where thousands are equal."""
    r = np.random.default_rng(V)
    combos = [(0, 1.0, 0.0), (3, 1.0, 0.0), (900, 1.0, 0.0), (0, 0.5, 0.0), (0, 1.0, 0.9), (50, 0.7, 0.2)]
    k, p, m = (np.array(x) for x in zip(*combos))
    for levels in (1, 3, 40):
        l = r.integers(0, levels, (len(combos), V)).astype(np.float32) * np.float32(0.25)
        check(l, r.random(len(combos)).astype(np.float32), None, k.astype(np.int32), p.astype(np.float32), m.astype(np.float32))


def test_signed_zeros_and_order():
    l = np.zeros((4, 300), np.float32)
    l[:, ::2] = -0.0  # equal to 0
    assert (check(l, [0.0, 0.0, 0.5, 0.999], None, [0, 1, 100, 100]) == [0, 0, 50, 99]).all()


def test_likeliest():
    """Temperature 0 or less, or NaN; top_k 1, top_p 0, min_p above 1: the first of the largest."""
    r = np.random.default_rng(0)
    l = r.integers(0, 50, (8, 20000)).astype(np.float32)
    want = l.argmax(1)
    u = np.full(8, 0.9999, np.float32)
    for kw in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=np.nan), dict(top_k=1), dict(top_p=0.0), dict(top_p=-1.0), dict(min_p=1.5)):
        tokens, probs = run_sample(l, u, **kw)
        assert np.array_equal(tokens, want) and (probs == 1).all(), kw
    assert np.array_equal(run_sample(l, u, temperature=0.0, top_k=5, top_p=0.5, min_p=0.1)[0], want)


def test_no_cut():
    """Cuts that cut nothing: top_k of the vocabulary or more, top_p from 1 on or NaN, min_p 0, below, or NaN."""
    r = np.random.default_rng(1)
    l = (r.standard_normal((6, 3000)) * 3).astype(np.float32)
    u = r.random(6).astype(np.float32)
    want = check(l, u)
    for kw in (dict(top_k=3000), dict(top_k=2**31 - 1), dict(top_k=-5), dict(top_p=1.5), dict(top_p=np.nan), dict(top_p=np.inf), dict(min_p=-1.0), dict(min_p=np.nan)):
        assert np.array_equal(run_sample(l, u, **kw)[0], want), kw


def test_masked():
    """-infinity has no weight; the type's lowest value hardly one; rows of -infinity alone, NaN or +infinity give none."""
    r = np.random.default_rng(2)
    V = 50000
    l = (r.standard_normal((8, V)) * 2).astype(np.float32)
    l[0, r.random(V) < 0.999] = -np.inf
    l[1, :] = -np.inf
    l[1, 31234] = -3.0
    l[2, r.random(V) < 0.99] = np.finfo(np.float32).min
    l[3, :] = -np.inf
    l[4, 7] = np.nan
    l[5, 49999] = np.inf
    l[6, :] = np.finfo(np.float32).min
    l[7, :-1] = -np.inf
    u = np.array([0.7, 0.3, 0.9, 0.5, 0.5, 0.5, 0.4, 0.2], np.float32)
    t = check(l, u)
    assert t[1] == 31234 and (t[3:6] == -1).all() and t[7] == V - 1
    for kw in (dict(top_k=2000), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=0.0), dict(top_k=40, top_p=0.9, min_p=0.01)):
        check(l, u, **kw)


def test_random_numbers():
    """The ends of [0, 1), and what lies outside."""
    r = np.random.default_rng(3)
    u = np.array([0.0, -0.0, -1.0, np.nan, np.nextafter(np.float32(1), np.float32(0)), 1.0, 7.0, np.inf, 1e-30], np.float32)
    l = np.tile((r.standard_normal(30000) * 2).astype(np.float32), (len(u), 1))
    for kw in ({}, dict(top_k=100), dict(top_p=0.8), dict(min_p=0.1)):
        tokens = check(l, u, **kw)
        assert (tokens[:4] == l[0].argmax()).all() and tokens[5] == tokens[6] == tokens[7]


@pytest.mark.parametrize("t", [1e-38, 1e-6, 0.01, 50.0, 1e10, 3e38, np.inf])
def test_temperatures(t):
    r = np.random.default_rng(4)
    for scale in (1.0, 1e4, 1e30):
        l = (r.standard_normal((4, 9000)) * scale).astype(np.float32)
        check(l, r.random(4).astype(np.float32), np.float32(t), [0, 50, 0, 0], [1.0, 1.0, 0.5, 1.0], [0.0, 0.0, 0.0, 0.3])


@pytest.mark.parametrize("V", [100, 16385, 33000])
def test_rows_apart(V):
    r = np.random.default_rng(5)
    l = (r.standard_normal((5, V)) * 2).astype(np.float32)
    u = r.random(5).astype(np.float32)
    want = check(l, u, top_k=30)
    for row in (V + 1, V + 6):
        assert np.array_equal(run_sample(l, u, top_k=30, row=row)[0], want)
    assert np.array_equal(run_sample(l, u, top_k=30, probs=False)[0], want)
    assert run_sample(np.zeros((0, V), np.float32), [])[0].size == 0


def test_drawn_often():
    """Many draws of one row come as often as their probabilities say (five standard deviations)."""
    V, n = 50, 4000
    r = np.random.default_rng(6)
    row = (r.standard_normal(V) * 1.5).astype(np.float32)
    tokens, _ = run_sample(np.tile(row, (n, 1)), r.random(n).astype(np.float32), temperature=0.8)
    p = np.exp(row.astype(np.float64) / np.float32(0.8))
    p /= p.sum()
    got = np.bincount(tokens, minlength=V)
    assert (np.abs(got - n * p) <= 5 * np.sqrt(n * p * (1 - p)) + 1).all()


def test_streams_and_graphs():
    """Calls under way together with their own workspaces; a captured one launched again over other logits and numbers."""
    r = np.random.default_rng(7)
    R, V = 3, 40000
    made = []
    for i in range(3):
        s, g = C.c_void_p(), C.c_void_p()
        kc.call("kcStreamCreate", C.byref(s))
        b = dict(logits=kc.Buffer(4 * R * V), u=kc.Buffer(4 * R), top_k=up([0, 40, 0], np.int32), top_p=up([1.0, 1.0, 0.9], np.float32))
        o = dict(tokens=Out(R, np.int32), probs=Out(R, np.float32))
        part = kc.Buffer(kc.sample_rows_part_bytes(R, V))
        args = kc.SampleRowsArgs(**{k: x.ptr for k, x in {**b, **o}.items()}, part=part.ptr, row=V, rows=R, n_vocab=V)
        kc.call("kcStreamBeginCapture", s)
        kc.launch("sample_rows", args, s)
        kc.call("kcStreamEndCapture", s, C.byref(g))
        made.append((s, g, b, o, part))
    for step in range(3):
        want = []
        for s, g, b, o, part in made:
            l, u = (r.standard_normal((R, V)) * 2).astype(np.float32), r.random(R).astype(np.float32)
            b["logits"].upload(l)
            b["u"].upload(u)
            want.append([plain_sample(l[i], u[i], 1.0, (0, 40, 0)[i], (1.0, 1.0, 0.9)[i])[0] for i in range(R)])
        for s, g, *_ in made:
            kc.call("kcGraphLaunch", g, s)
        kc.synchronize()
        for (s, g, b, o, part), w in zip(made, want):
            got = o["tokens"].buf.download(np.int32, R, 256)
            assert all(got[i] in w[i] for i in range(R)), step
    for s, g, b, o, part in made:
        kc.call("kcGraphDestroy", g)
        kc.call("kcStreamDestroy", s)
        o["tokens"].get(), o["probs"].get()
        for x in [part, *b.values()]:
            x.free()
