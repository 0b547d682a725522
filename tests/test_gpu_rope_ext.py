"""rope_ext against its definition in 64 bits (tests/serve.py derives the bounds)."""
import numpy as np
import pytest

import kernelcore_amd as kc
from tests.serve import Out, plain_turn, up

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def runtime():
    kc.init()
    yield
    kc.synchronize()


def strided(r, n, heads, D, row, head):
    """(array [n][heads][D], flat memory with these strides in values)"""
    x = r.standard_normal((n, heads, D)).astype(np.float32)
    flat = np.full(max(1, (n - 1) * row + (heads - 1) * head + D), np.nan, np.float32)
    view = np.lib.stride_tricks.as_strided(flat, x.shape, (4 * row, 4 * head, 4))
    view[...] = x
    return x, flat


def run(N, H, K, D, n_rot, inter, pos=None, slots=None, rows=None, scale=1.0, pad=0, q=True, k=True, v=True, in_place=False, base=1e6, outer=False,
        misalign=0):
    r = np.random.default_rng([N, H, D, n_rot])
    pos = r.integers(0, 200000, N) if pos is None else np.asarray(pos)
    rows = N + 9 if rows is None else rows
    slots = r.permutation(rows)[:N] if slots is None else np.asarray(slots)
    freqs, _ = kc.rope_freqs(n_rot, base)
    qh, kh = D + pad, D + 2 * pad
    qr, kr = H * qh + pad, K * kh + 3 * pad
    xq, fq = strided(r, N, H, D, qr, qh)
    xk, fk = strided(r, N, K, D, kr, kh)
    xv, fv = strided(r, N, K, D, kr, kh)
    ch = 2 * (D + pad) if not outer else 2 * (D + pad) * rows  # bytes between heads of a cache row
    crow = (K * ch + 2 * pad) if not outer else 2 * (D + pad)
    size = ((rows - 1) * crow + (K - 1) * ch + 2 * D) // 2
    before = np.arange(size, dtype=np.uint16)
    ins = dict(pos=up(pos, np.int32), freqs=up(freqs, np.float64), slots=up(slots, np.int64))
    shift = 4 * misalign
    bufs = {}
    for name, f, have in (("q", fq, q), ("k", fk, k), ("v", fv, v and k)):
        if have:
            bufs[name] = kc.Buffer(f.nbytes + 64)
            bufs[name].upload(f, shift)
            ins[name] = type("P", (), {"ptr": bufs[name].ptr + shift})
    oh, orow = (qh, qr) if in_place else (D + pad, H * (D + pad) + 5 * pad)
    osize = max(1, (N - 1) * orow + (H - 1) * oh + D)
    o = {}
    if q:
        o["q_out"] = Out(osize, np.float32, np.full(osize, 7.0)) if not in_place else None
    if k:
        o["k_cache"] = Out(size, np.uint16, before)
        if v:
            o["v_cache"] = Out(size, np.uint16, before)
    ptr = {n: (x.ptr if x else ins["q"].ptr) for n, x in o.items()}
    kc.launch("rope_ext", kc.RopeExtArgs(**{n: b.ptr for n, b in ins.items()}, **ptr, n_tokens=N, H=H, H_kv=K, D=D, n_rot=n_rot, interleaved=int(inter),
                                         q_tok=qr, q_head=qh, k_tok=kr, k_head=kh, v_tok=kr, v_head=kh, out_tok=orow, out_head=oh, cache_rows=rows,
                                         kc_row=crow, kc_head=ch, vc_row=crow, vc_head=ch, scale=scale))
    kc.synchronize()
    if q:
        if in_place:
            flat = bufs["q"].download(np.float32, fq.size, shift)
            rest = fq.copy()
        else:
            flat, rest = o["q_out"].get(), np.full(osize, 7.0, np.float32)
        st = (4 * orow, 4 * oh, 4)
        got = np.lib.stride_tricks.as_strided(flat, (N, H, D), st).copy()
        want, bound = plain_turn(xq, pos, freqs, scale, n_rot, inter)
        assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) - bound).max())
        np.lib.stride_tricks.as_strided(rest, (N, H, D), st)[...] = got
        assert np.array_equal(flat.view(np.uint32), rest.view(np.uint32))  # nothing between the rows
    last = {}  # of tokens with the same slot the last one
    for t, s in enumerate(slots):
        if 0 <= s < rows:
            last[int(s)] = t
    for name, x in (("k_cache", xk), ("v_cache", xv)):
        if name not in o:
            continue
        flat, rest = o[name].get(), before.copy()
        st = (crow, ch, 2)
        got, old = (np.lib.stride_tricks.as_strided(y, (rows, K, D), st) for y in (flat, rest))
        want, bound = plain_turn(x, pos, freqs, scale, n_rot, inter) if name == "k_cache" else (x.astype(np.float64), np.zeros(x.shape))
        for s, t in last.items():
            g = got[s].view(np.float16).astype(np.float64)
            # half a step of fp16 (2^-11, subnormal 2^-25) and the bound
            assert (np.abs(g - want[t]) <= bound[t] * 1.001 + np.maximum(np.abs(want[t]) * 2.0 ** -11, 2.0 ** -25) + 2.0 ** -40).all(), (name, s)
            if name == "v_cache":
                assert np.array_equal(got[s], x[t].astype(np.float16).view(np.uint16))
            old[s] = got[s]
        assert np.array_equal(flat, rest), name  # every other row as it was
    for b in list(bufs.values()) + [ins["pos"], ins["freqs"], ins["slots"]]:
        b.free()


SHAPES = [(1, 32, 8, 128, 128), (8, 24, 8, 128, 64), (5, 1, 1, 64, 64), (3, 8, 2, 256, 256), (7, 3, 3, 80, 32), (4, 2, 1, 96, 96), (2, 5, 5, 64, 10),
          (3, 2, 2, 64, 2), (2, 1, 1, 2, 2), (3, 4, 2, 6, 4), (2, 2, 1, 1024, 1024), (2, 2, 2, 1000, 998), (700, 4, 2, 128, 128), (1300, 2, 1, 64, 32)]


@pytest.mark.parametrize("inter", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("N,H,K,D,n_rot", SHAPES)
def test_shapes(N, H, K, D, n_rot, inter):
    print("rope_ext", N, H, K, D, n_rot, inter, flush=True)
    run(N, H, K, D, n_rot, inter)


@pytest.mark.parametrize("inter", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("kw", [dict(pad=3), dict(pad=1, misalign=1), dict(in_place=True), dict(in_place=True, pad=5), dict(k=False), dict(v=False), dict(q=False),
                                dict(scale=1.3465735), dict(scale=-0.5), dict(outer=True), dict(outer=True, pad=1), dict(base=1.5)], ids=str)
def test_layouts(inter, kw):
    print("rope_ext", inter, kw, flush=True)
    run(37, 6, 3, 72, 48, inter, **kw)


@pytest.mark.parametrize("inter", [False, True], ids=["halves", "pairs"])
def test_far_positions(inter):
    run(8, 4, 2, 128, 128, inter, pos=[0, 1, 131071, 2**20 + 1, 2**24 + 1, 2**30 + 12345, 2**31 - 1, 2**31 - 2])


def test_no_token():
    run(0, 4, 2, 64, 64, False, rows=4, slots=np.zeros(0, np.int64))


@pytest.mark.parametrize("N", [6, 40, 3000])
def test_slots(N):
    """Slots outside the cache store nothing; of tokens with the same slot the last one is stored."""
    r = np.random.default_rng(N)
    rows = 64
    slots = r.integers(0, rows, N)
    slots[::5] = r.choice(np.array([-1, -2**40, rows, 2**32, 2**32 + 3, 2**62]), len(slots[::5]))
    run(N, 2, 2, 64, 32, False, rows=rows, slots=slots)


def test_special_values():
    """Infinities and NaN stay where they are; values past fp16's range become infinities."""
    n, D = 2, 64
    v = np.array([np.inf, -np.inf, np.nan, 70000.0, -65519.9, 65520.0, -0.0, 1e-8], np.float32)
    x = np.tile(v, (n, 1, D // 8)).astype(np.float32)
    freqs, _ = kc.rope_freqs(D, 1e4)
    b = dict(k=up(x, np.float32), v=up(x, np.float32), pos=up([0, 0], np.int32), freqs=up(freqs, np.float64), slots=up([1, 0], np.int64))
    kcache, vcache = Out(n * D, np.uint16), Out(n * D, np.uint16)
    kc.launch("rope_ext", kc.RopeExtArgs(**{a: y.ptr for a, y in b.items()}, k_cache=kcache.ptr, v_cache=vcache.ptr, n_tokens=n, H_kv=1, D=D, n_rot=D, k_tok=D,
                                         k_head=D, v_tok=D, v_head=D, cache_rows=n, kc_row=2 * D, kc_head=2 * D, vc_row=2 * D, vc_head=2 * D, scale=1.0))
    kc.synchronize()
    kcache.get()
    got = vcache.get().view(np.float16).reshape(n, D)
    with np.errstate(over="ignore"):
        want = x[:, 0].astype(np.float16)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])
