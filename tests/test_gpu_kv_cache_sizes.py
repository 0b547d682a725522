"""kv_keep and set_rows_q4_0 at the sizes where another form of their kernels takes over, and between them: bits against plain forms."""
import numpy as np
import pytest

import kernelcore_amd as kc
from tests.test_gpu_kv_cache import plain_keep, store

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def runtime():
    kc.init()
    yield
    kc.synchronize()


# rows held in registers up to 4096, 16384 and 32768 positions, then read by each sweep
@pytest.mark.parametrize("T,n_keep,first,recent", [(4096, 1000, 4, 64), (4097, 1000, 4, 64), (4097, 4096, 1, 0), (6001, 3001, 77, 1001), (16384, 2048, 4, 256),
                                                   (16385, 2048, 4, 256), (16384, 16383, 0, 0), (20011, 777, 13, 301), (32768, 4096, 4, 256), (32768, 1, 0, 0),
                                                   (32769, 4096, 4, 256), (40013, 20000, 1023, 65)])
@pytest.mark.parametrize("kind", ["random", "ties", "special"])
def test_keep(T, n_keep, first, recent, kind):
    heads = 2
    r = np.random.default_rng([T, n_keep])
    w = (r.random((heads, T)) ** 8 * 10).astype(np.float32)
    if kind == "ties":
        w = r.integers(0, 3, (heads, T)).astype(np.float32)
    if kind == "special":
        w = r.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1.0, 3e38], np.float32), (heads, T))
    row, krow = T + 3, n_keep + 5
    wide = np.full((heads, row), 1e9, np.float32)
    wide[:, :T] = w
    bw, bk = kc.Buffer.of(wide), kc.Buffer.of(np.full(heads * krow + 16, -7, np.int32))
    kc.launch("kv_keep", kc.KvKeepArgs(bw.ptr, bk.ptr, heads, T, row, n_keep, krow, first, recent))
    want = np.full(heads * krow + 16, -7, np.int32)
    want[:heads * krow].reshape(heads, krow)[:, :n_keep] = plain_keep(w, n_keep, first, recent)
    assert np.array_equal(bk.download(np.int32), want)
    bw.free(), bk.free()


# one, two and eight rows to a workgroup: up to 2048 rows, up to 8192 and beyond
@pytest.mark.parametrize("n,rows", [(96, 2048), (96, 2049), (1056, 2050), (32, 5001), (32, 8192), (32, 8193), (1056, 8197), (32, 20007)])
@pytest.mark.parametrize("how", ["each", "repeated", "neighbours"])
def test_store(n, rows, how):
    r = np.random.default_rng([n, rows])
    x = r.standard_normal((rows, n)).astype(np.float32)
    cache = rows + 40
    idx = r.permutation(cache)[:rows].astype(np.int64)
    if how == "repeated":  # far apart: most rows are stored over
        idx = r.integers(-2, cache // 3, rows)
        idx[r.random(rows) < 0.05] = 1 << 32
        cache = cache // 3 - 1
    if how == "neighbours":  # within the rows of a workgroup and across two of them
        idx = np.arange(rows) // 3 * 2
        idx[rows - 5:] = idx[rows - 1]
    got, want = store(x, idx, cache)
    assert np.array_equal(got, want)
