"""flash_ext_* and attn_weights_* where their definition is easily missed, against plain forms in 64 bits (tests/kvcache.py)."""
import math

import numpy as np
import pytest

import kernelcore_amd as kc
from tests.kvcache import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def runtime():
    kc.init()
    yield
    kc.synchronize()


CACHES = pytest.mark.parametrize("q4", [False, True], ids=["f16", "q4_0"])
# one row tile and several on the few-rows kernel, then the many-rows kernel, of each head size, and in several ranges
ROWS = [(8, 2, 128, 1, 2000), (6, 2, 64, 5, 700), (4, 2, 256, 3, 333), (8, 2, 128, 60, 330), (32, 32, 64, 290, 450), (16, 16, 128, 300, 421),
        (16, 16, 256, 260, 501), (5, 1, 128, 700, 1111), (8, 2, 256, 330, 900)]


@CACHES
@pytest.mark.parametrize("H,K,D,N,T", ROWS)
@pytest.mark.parametrize("how", ["last", "ascending", "shuffled", "early", "outside", "prefix"])
def test_query_positions_alone(q4, H, K, D, N, T, how):
    """qpos stands in for pos0 + i, whatever pos0 is, where nothing else shapes the scores."""
    print(f"flash_ext q4={q4} H={H}/{K} D={D} N={N} T={T} {how}", flush=True)
    r = np.random.default_rng([N, T])
    spread = np.sort(r.integers(0, T, N))
    qpos, pos0 = {"last": (np.full(N, T - 1), 0), "ascending": (spread, 0), "shuffled": (r.permutation(spread), 3), "early": (spread // 3, T),
                  "outside": (np.where(np.arange(N) % 2 == 0, -1 - spread, T + spread), 0),  # (a negative one sees nothing)
                  "prefix": (spread // 2, T)}[how]
    c = Case(q4, H, K, D, N, T, qpos=qpos.astype(np.int32), pos0=pos0, prefix=T // 2 + 1 if how == "prefix" else 0)
    _, sums = c.check()
    if how in ("last", "outside"):  # and the weights of the same call
        lse = c.expected()[2].astype(np.float32)
        want, bound = c.expected_weights(lse, None, 0.0)
        assert (np.abs(c.weights(lse) - want) <= bound).all()


@CACHES
@pytest.mark.parametrize("H,K,D,T", [(4, 2, 64, 91), (8, 2, 128, 5000), (256, 2, 64, 8300)])
def test_mask_rows_far_apart(q4, H, K, D, T):
    """Mask rows 4 GiB apart, two of them, against packed ones: few rows in one range and in several, many rows."""
    r = np.random.default_rng(T)
    m = r.standard_normal((2, T + T % 2)).astype(np.float16)
    m[r.random(m.shape) < 0.4] = -np.inf
    c = Case(q4, H, K, D, 2, T, causal=0, mask=m)
    want, lse = c.attend()
    w_want = c.weights(lse)
    step = 4 << 30
    far = kc.Buffer(step + m[0].nbytes)
    for i in range(2):
        far.upload(m[i], i * step)
    b, d = c.upload(), c.dims(m_row=step // 4)
    out, part, w, bl = kc.Buffer(want.nbytes), kc.Buffer(kc.flash_ext_part_bytes(d) + 4), kc.Buffer(w_want.nbytes), kc.Buffer.of(lse)
    shape = dict(c.shape_args(b, d), mask=far.ptr)
    kc.launch(c.name("flash_ext"), kc.FlashExtArgs(v=b["v"].ptr, out=out.ptr, part=part.ptr, **shape))
    assert np.array_equal(out.download(np.float32).reshape(want.shape), want)
    kc.launch(c.name("attn_weights"), kc.AttnWeightsArgs(lse=bl.ptr, w=w.ptr, w_row=T, **shape))
    assert np.array_equal(w.download(np.float32).reshape(w_want.shape), w_want)
    for x in (far, out, part, w, bl, *b.values()):
        x.free()


def enlarge(c, name, at, head, factor):
    """The key or value rows `at` of a KV head, multiplied by a power of two."""
    a = getattr(c, name)
    if c.q4:
        d = a.reshape(c.T, c.K, -1, 18)[at, head, :, :2]
        a.reshape(c.T, c.K, -1, 18)[at, head, :, :2] = (np.ascontiguousarray(d).view(np.float16) * np.float16(factor)).view(np.uint8)
    else:
        a[at, head] *= np.float16(factor)


@CACHES
@pytest.mark.parametrize("H,K,D,N,T", ROWS)
def test_a_cap_keeps_rows_and_keys_apart(q4, H, K, D, N, T):
    """Under a cap a score's bits depend on its own query and key: not on keys that the query does not see, nor on other queries,
    however large (their tanh takes another form)."""
    r = np.random.default_rng(N)
    c = Case(q4, H, K, D, N, T, cap=20.0)
    at, few = T - max(1, N // 2), N == 1
    if few:  # hidden by a mask
        at = T // 2
        c.mask = np.zeros((1, T + T % 2), np.float16)
        c.mask[0, at] = -np.inf
    clean, sums = c.check()
    lse = c.expected()[2].astype(np.float32)
    weights = c.weights(lse)
    enlarge(c, "k", at, 0, 1024)
    got, got_sums = c.check()
    hidden = np.arange(N) + T - N < at if not few else np.array([True])
    assert hidden.any()
    assert np.array_equal(got[hidden], clean[hidden]) and np.array_equal(got_sums[hidden], sums[hidden])
    others = np.arange(T) != at
    assert np.array_equal(c.weights(lse)[:, others], weights[:, others])
    if N > 1:
        c = Case(q4, H, K, D, N, T, cap=20.0)
        c.q[N // 2] *= 1024
        got, got_sums = c.check()
        rest = np.arange(N) != N // 2
        assert np.array_equal(got[rest], clean[rest]) and np.array_equal(got_sums[rest], sums[rest])


@CACHES
@pytest.mark.parametrize("spread", [1.0, 8.0])
def test_caps_among_the_scores(q4, spread):
    """Scores on both sides of the border between the forms of tanh."""
    for N, T in ((1, 500), (40, 300), (1100, 200)):
        Case(q4, 8, 2, 128, N, T, cap=2.0, spread=spread).check()


class Infinite(Case):
    """Keys with infinities and NaN: a score of -infinity has weight 0, one of +infinity or NaN makes the query's result NaN."""

    def scores(self):
        x, seen, terms = super().scores()
        return np.where(np.isneginf(x), -np.inf, x), seen & ~np.isneginf(x), np.where(np.isfinite(terms), terms, self.cap)

    def check(self):
        out, sums = self.attend()
        x, seen, _ = self.scores()
        lost = (seen & ~np.isfinite(x)).any(-1)
        with np.errstate(invalid="ignore", over="ignore"):
            want, bound, lse, lse_bound = self.expected()
            lse32 = np.where(lost, 0.0, lse).astype(np.float32)
            w_in = np.random.default_rng(1).random((self.K, self.T)).astype(np.float32)
            w, w_bound = self.expected_weights(lse32, w_in, 0.5)
        assert np.isnan(out[lost]).all() and np.isnan(sums[lost]).all()
        kept = ~lost
        assert (np.abs(out[kept] - want[kept]) <= bound[kept]).all()
        assert (np.isneginf(sums[kept]) == np.isneginf(lse[kept])).all()
        fin = kept & np.isfinite(lse)
        assert (np.abs(sums[fin] - lse[fin]) <= lse_bound[fin]).all()
        got = self.weights(lse32, w_in, 0.5)
        assert (np.isnan(got) == np.isnan(w)).all()
        plain = np.isfinite(w)
        assert (np.abs(got[plain] - w[plain]) <= w_bound[plain]).all() and (np.isinf(got) == np.isinf(w)).all()
        return lost


@CACHES
@pytest.mark.parametrize("H,K,D,N,T", ROWS + [(32, 32, 64, 1, 2300), (32, 8, 128, 9, 4201), (16, 16, 256, 2, 4300)])  # (weights: walks over the keys)
@pytest.mark.parametrize("cap", [0.0, 15.0])
def test_infinities_and_nan_in_seen_keys(q4, H, K, D, N, T, cap):
    print(f"flash_ext q4={q4} H={H}/{K} D={D} N={N} T={T} cap={cap}", flush=True)
    r = np.random.default_rng([N, T])
    c = Infinite(q4, H, K, D, N, T, cap=cap, causal=0)
    # q of every token: the values that meet the infinity positive (whose low parts are 0 or negative for some) or, of KV head 0's
    # first query head, too small beside the others to be fp16 numbers
    at = 35
    c.q[:, :, 32:64] = np.abs(c.q[:, :, 32:64])
    c.q[:, 0, at] = 1e-30
    rows = sorted(set([0, T // 3, T - 1]))
    for j in rows:
        if q4:  # every product of the block negative: codes below 8
            b = c.k.reshape(T, K, -1, 18)[j]
            b[:, 1, :2] = np.frombuffer(np.float16(np.inf).tobytes(), np.uint8)
            b[:, 1, 2:] = r.integers(0, 8, (K, 16)) + 16 * r.integers(0, 8, (K, 16))
        else:
            c.k[j, :, at] = -np.inf
    lost = c.check()
    assert not lost.any()
    j = rows[len(rows) // 2]
    m = np.zeros((N, T + T % 2), np.float16)
    m[N // 2:, j] = -np.inf
    if N == 1:
        m[:] = 0
    c.mask = m
    for bad in (np.inf, np.nan):
        if q4:
            b = c.k.reshape(T, K, -1, 18)[j]
            b[K - 1, 0, :2] = np.frombuffer(np.float16(bad).tobytes(), np.uint8)
            b[K - 1, 0, 2:] = np.arange(16) * 17  # (a code of 8: 0 times infinity)
        else:
            c.k[j, K - 1, 7] = bad
        lost = c.check()
        seen = np.arange(N) < N // 2 if N > 1 else np.ones(1, bool)
        assert not lost[~seen].any() and (np.isinf(bad) or lost[seen][:, (K - 1) * H // K:].all())


@CACHES
def test_zero_times_an_infinity(q4):
    """A zero of q that meets an infinity, and a scale of zero: NaN, for the queries that see the key."""
    for N, T in ((1, 200), (40, 200), (1100, 200)):
        c = Infinite(q4, 8, 2, 128, N, T)
        c.q[:, 3, 40] = 0
        if q4:
            b = c.k.reshape(T, 2, -1, 18)[0, 0, 1]
            b[:2] = np.frombuffer(np.float16(np.inf).tobytes(), np.uint8)
            b[2:] = 0x11
            c.q[:, :, 32:64] = np.abs(c.q[:, :, 32:64])
        else:
            c.q[:, :3, 40] = np.abs(c.q[:, :3, 40])
            c.k[0, 0, 40] = -np.inf
        lost = c.check()
        assert lost[:, 3].all() and not lost[:, :3].any() and not lost[:, 4:].any()
        c.scale = 0.0
        assert c.check()[:, :4].all()


@CACHES
@pytest.mark.parametrize("H,K,D,N,T", [(8, 2, 128, 1, 333), (8, 2, 64, 40, 333), (16, 16, 256, 260, 501)])
def test_caps_of_any_size(q4, H, K, D, N, T):
    """The smallest cap (every score 0 beside it, NaN in none) and the largest (no cap), with q of any size."""
    for cap in (2.0 ** -100, 2.0 ** -20, 2.0 ** 30, 2.0 ** 100):
        for spread, scale in ((1.0, 1.0 / math.sqrt(D)), (1e30, 1e-31), (1e30, 1.0), (1e-30, 1e30)):
            c = Case(q4, H, K, D, N, T, cap=cap, spread=spread, scale=scale)
            c.q[0, 0] = 0
            if q4:  # (and a score of 0 beside q of any size)
                c.k.reshape(T, K, -1, 18)[1, ..., :2] = 0
            else:
                c.k[1] = 0
            if cap < 1 or scale * spread <= 1:
                c.check()


@CACHES
@pytest.mark.parametrize("H,K,N,T", [(8, 2, 12, 400), (16, 16, 60, 200), (8, 2, 40, 300), (16, 16, 90, 1000), (16, 16, 90, 2500)])
@pytest.mark.parametrize("shape", ["plain", "cap_bias", "kept"])
def test_weights_of_heads_of_256(q4, H, K, N, T, shape):
    """Two, eight and four wavefronts to a key tile, four to four, with and without positions of the keys' own."""
    r = np.random.default_rng(T)
    kw = dict(cap=10.0, bias=True, prefix=T // 3) if shape == "cap_bias" else {}
    if shape == "kept":
        kpos = np.sort(r.choice(3 * T + 1, (K, T)), axis=1).astype(np.int32)
        kpos[r.random((K, T)) < 0.2] = -1
        kw = dict(kpos=kpos, pos0=2 * T, bias=True)
    c = Case(q4, H, K, 256, N, T, **kw)
    lse = c.expected()[2].astype(np.float32)
    w_in = r.random((K, T)).astype(np.float32)
    want, bound = c.expected_weights(lse, w_in, 0.75)
    assert (np.abs(c.weights(lse, w_in, 0.75) - want) <= bound).all()


@CACHES
@pytest.mark.parametrize("H,K,D,N,T", [(4, 2, 256, 3, 200), (16, 16, 256, 260, 501), (6, 2, 64, 5, 200), (32, 32, 64, 290, 450)])
def test_infinities_in_values(q4, H, K, D, N, T):
    """An infinite or NaN value: just its own column (of a 4-bit cache, its block's), for the queries that see it."""
    c = Case(q4, H, K, D, N, T)
    clean, sums = c.attend()
    at = T - N // 2 - 1
    if q4:
        c.v.reshape(T, K, -1, 18)[at, 1, 1, :2] = np.frombuffer(np.float16(-np.inf).tobytes(), np.uint8)
        cols = np.arange(32, 64)
    else:
        c.v[at, 1, [1, D - 2]] = np.nan, np.inf
        cols = np.array([1, D - 2])
    got, got_sums = c.attend()
    hidden = np.arange(N) + T - N < at
    others = np.setdiff1d(np.arange(D), cols)
    assert np.array_equal(got[hidden], clean[hidden]) and np.array_equal(got[..., others], clean[..., others]) and np.array_equal(got_sums, sums)
    G = H // K
    assert np.array_equal(got[:, :G], clean[:, :G]) and np.array_equal(got[:, 2 * G:], clean[:, 2 * G:])
    assert not np.isfinite(got[~hidden][:, G:2 * G][..., cols]).any()
