"""kv_pages on trees of many nodes and great depth: more than a launch takes, sequences that begin and end anywhere."""
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


def check(have, add, parent, words):
    """Everything but positions and trees as without trees; those from each node's parent's."""
    page, n = 16, int(np.sum(add))
    need = int((-(-(np.asarray(have) + add) // page) - -(-np.asarray(have) // page)).sum())
    free = np.random.default_rng(0).permutation(need).astype(np.int32)
    table = np.full((len(add), int((-(-(np.asarray(have) + add) // page)).max())), 5, np.int32)
    got = run_pages(have, add, free, table, page, n, parent, words)
    want = plain_pages(have, add, free, table, page, n)
    tree, pos = np.zeros((n, words), np.uint32), np.zeros(n, np.int64)
    t0 = 0
    for h, a in zip(have, add):
        for i in range(a):
            up = int(parent[t0 + i])
            pos[t0 + i] = h
            if 0 <= up < i:
                tree[t0 + i], pos[t0 + i] = tree[t0 + up], pos[t0 + up] + 1
            if i < 32 * words:
                tree[t0 + i, i >> 5] |= np.uint32(1 << (i & 31))
        t0 += a
    want.update(tree=tree.view(np.int32), pos=np.minimum(pos, 2**31 - 1).astype(np.int32))
    for k in want:
        assert np.array_equal(got[k], want[k]), (k, np.argwhere(got[k] != want[k])[:4].tolist())


def trees(r, add, kind):
    parent = []
    for n in add:
        i = np.arange(n)
        parent.append(dict(chain=i - 1, near=i - 1 - np.minimum(r.integers(0, 4, n), i), random=(r.random(n) * i).astype(int) - (i == 0),
                           wild=np.where(r.random(n) < 0.02, r.choice([-1, -7, n, 2**31 - 1], n), i - 1 - r.integers(0, 40, n)))[kind])
    return np.concatenate(parent)


@pytest.mark.parametrize("words", [1, 2, 3, 64])
@pytest.mark.parametrize("kind", ["chain", "near", "random", "wild"])
@pytest.mark.parametrize("add", [[2048], [100, 20000, 300, 7]], ids=str)
def test_deep(words, kind, add):
    print("kv_pages", add, kind, words, flush=True)
    r = np.random.default_rng([words, len(add), add[0]])
    check(r.integers(0, 100, len(add)), add, trees(r, add, kind), words)


LAUNCH = 1 << 18


@pytest.mark.parametrize("words", [1, 3, 64])
@pytest.mark.parametrize("kind", ["chain", "near", "wild"])
@pytest.mark.parametrize("add", [[LAUNCH - 68, 64, 64, 64, 200], [30, LAUNCH + 500, 7]], ids=str)
def test_several_launches(words, kind, add):
    """A tree's nodes of a launch after the one that its root is in; one that begins with a launch."""
    print("kv_pages", add, kind, words, flush=True)
    r = np.random.default_rng([words, len(add), add[0]])
    check(r.integers(0, 100, len(add)), add, trees(r, add, kind), words)


@pytest.mark.parametrize("words", [1, 2])
def test_short_trees(words):
    """Trees of a few nodes on both sides of a launch's end."""
    r = np.random.default_rng(words)
    add = r.integers(1, 60, 10000)
    check(r.integers(0, 100, len(add)), add, trees(r, add, "random"), words)


def test_deep_far():
    """Positions past the largest number stay there, in every launch."""
    n = LAUNCH + 7000
    have, page = 2**31 - LAUNCH - 300, 65536
    got = run_pages([have], [n], np.zeros(1, np.int32), np.zeros((1, 1), np.int32), page, n, np.arange(n) - 1, 1)
    assert np.array_equal(got["pos"], np.minimum(have + np.arange(n, dtype=np.int64), 2**31 - 1)) and (got["slots"] == -1).all() and got["len"] == 2**31 - 1
