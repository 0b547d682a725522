"""sample_rows where the random number is 1 or more, which counts as the largest double below 1: the draw ends at the last token that is kept
and has weight. Many rows each, as it takes a rounding in the sums to go past it (one row in a hundred and less)."""
import numpy as np
import pytest

import kernelcore_amd as kc
from tests.serve import run_sample

pytestmark = pytest.mark.gpu

EPS = np.longdouble(2.0 ** -40)  # of the whole: what a border may be off by (tests/serve.py, plain_sample)


@pytest.fixture(scope="module", autouse=True)
def runtime():
    kc.init()
    yield
    kc.synchronize()


def right(l, u, token, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Whether the definition, with each border moved by up to EPS, draws this token."""
    order = np.argsort(-l.astype(np.float64), kind="stable")
    at = np.flatnonzero(order == token)
    if at.size == 0:
        return False
    at = int(at[0])
    z = l[order].astype(np.longdouble) / np.longdouble(np.float32(temperature))
    w = np.where(np.isneginf(l[order]), np.longdouble(0), np.exp(np.where(np.isneginf(l[order]), 0, z - z[0])))
    finite = int(np.isfinite(l).sum())
    k = min(top_k, finite) if top_k > 0 else finite
    c = np.cumsum(w)
    u = np.longdouble(min(1.0, float(u)))
    for cut in (0, EPS, -EPS):
        m = k
        if top_p < 1:
            m = min(m, int((c[:k] < np.longdouble(np.float32(top_p)) * c[k - 1] * (1 + cut)).sum()) + 1)
        if min_p > 0:
            m = min(m, max(1, int((w >= np.longdouble(np.float32(min_p)) * (1 + cut)).sum())))
        last = int(np.flatnonzero(w[:m] > 0)[-1])
        if at > last:
            continue
        whole = c[m - 1]
        if (at == 0 or c[at - 1] <= (u + EPS) * whole) and (c[at] > (u - EPS) * whole or at == last):
            return True
    return False


def check(l, temperature, top_k=None, top_p=None, min_p=None, us=(1.0, 7.0, np.nextafter(np.float32(1), np.float32(0)))):
    R = len(l)
    u = np.resize(np.array(us, np.float32), R)
    tokens, probs = run_sample(l, u, temperature, top_k, top_p, min_p)
    one = lambda x, r, d: d if x is None else x[r].item()  # noqa: E731
    wrong = [(r, int(tokens[r]), float(u[r])) for r in range(R)
             if not right(l[r], u[r], tokens[r], temperature[r], one(top_k, r, 0), one(top_p, r, 1.0), one(min_p, r, 0.0))]
    assert not wrong, (len(wrong), wrong[:5])
    assert (probs > 0).all()


def rows_of(r, R, V, far):
    """Rows of every spread from flat on, some in steps; with `far`, half of the logits where weights are about 2^-63 of the largest."""
    spread = r.choice([0.0, 1e-4, 0.01, 0.3, 1.0, 2.5, 5.0], R)
    l = r.standard_normal((R, V)) * spread[:, None]
    l[::3] = np.round(l[::3] * 4) / 4
    if far:
        l = np.where(r.random((R, V)) < 0.5, -43.5 - r.random((R, V)), l)
        l[:, 0] = 0.0
    return l.astype(np.float32), np.where(r.random(R) < 0.5, 1.0, r.uniform(0.3, 1.8, R)).astype(np.float32)


@pytest.mark.parametrize("V,R", [(7, 1500), (100, 1500), (399, 1500), (3000, 400), (40000, 60)])
@pytest.mark.parametrize("far", [False, True])
def test_no_cut(V, R, far):
    print("sample_rows", V, R, far, flush=True)
    l, t = rows_of(np.random.default_rng([V, far]), R, V, far)
    check(l, t)


@pytest.mark.parametrize("V,R", [(7, 1500), (100, 1500), (399, 1500), (3000, 400), (40000, 60)])
@pytest.mark.parametrize("cut", ["top_k", "top_p", "min_p", "all"])
def test_cuts(V, R, cut):
    """The last token that a cut keeps, whose bin holds tokens that it does not keep, and bins without tokens behind it."""
    print("sample_rows", V, R, cut, flush=True)
    r = np.random.default_rng([V, len(cut), cut[-1] == "k"])
    l, t = rows_of(r, R, V, False)
    k = r.integers(1, V + 1, R).astype(np.int32) if cut in ("top_k", "all") else None
    p = r.uniform(0.05, 0.999, R).astype(np.float32) if cut in ("top_p", "all") else None
    m = r.uniform(0.001, 0.4, R).astype(np.float32) if cut in ("min_p", "all") else None
    check(l, t, k, p, m)
