"""set_rows_q4_0 / get_rows_q4_0, kv_keep and kv_gather: bits against plain forms in exact arithmetic."""
import numpy as np
import pytest

import kernelcore_amd as kc
from tests.kvcache import pack_q4, unpack_q4

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def runtime():
    kc.init()
    yield
    kc.synchronize()


def store(x, idx, dst_rows, src_row=None, dst_row=None, fill=0xA5):
    rows, n = x.shape
    src_row, dst_row = src_row or n, dst_row or n // 32 * 18
    src = np.full(max(1, (rows - 1) * src_row + n), 3.0, np.float32)
    for r in range(rows):
        src[r * src_row:r * src_row + n] = x[r]
    dst = np.full(max(1, dst_rows) * dst_row + 64, fill, np.uint8)
    bs, bi, bd = kc.Buffer.of(src), kc.Buffer.of(np.asarray(idx, np.int64)), kc.Buffer.of(dst)
    kc.launch("set_rows_q4_0", kc.SetRowsQ40Args(bs.ptr, bi.ptr, bd.ptr, n, rows, src_row, dst_rows, dst_row))
    got = bd.download(np.uint8)
    want = dst.copy()
    b = pack_q4(x)
    for r, at in enumerate(idx):  # (in order: the last of equal indices stays)
        if 0 <= at < dst_rows:
            want[at * dst_row:at * dst_row + n // 32 * 18] = b[r]
    for x_ in (bs, bi, bd):
        x_.free()
    return got, want


@pytest.mark.parametrize("n,rows", [(32, 1), (64, 1), (1024, 1), (1056, 3), (128, 64), (128, 65), (96, 300), (2048, 130), (4096, 9)])
def test_store(n, rows):
    r = np.random.default_rng([n, rows])
    x = (r.standard_normal((rows, n)) * 10.0 ** r.integers(-3, 3, (rows, 1))).astype(np.float32)
    got, want = store(x, r.permutation(rows + 5)[:rows], rows + 5)
    assert np.array_equal(got, want)
    got, want = store(x, r.permutation(rows + 5)[:rows], rows + 5, src_row=n + 7, dst_row=n // 32 * 18 + 6)
    assert np.array_equal(got, want)


@pytest.mark.parametrize("rows", [7, 200])
def test_store_indices(rows):
    """Indices outside the cache (as 64-bit values), and the same index several times: the last row stays."""
    r = np.random.default_rng(rows)
    x = r.standard_normal((rows, 64)).astype(np.float32)
    idx = r.integers(0, 5, rows)
    idx[rows // 2] = -1
    idx[rows // 3] = 1 << 32
    idx[rows // 4] = 5
    got, want = store(x, idx, 5)
    assert np.array_equal(got, want)


def test_store_borders():
    """Values on and next to the borders between codes, equal magnitudes of both signs, zeros, subnormals, blocks that hold
    an infinity or NaN, scales beyond fp16."""
    rows = []
    for d in (1.0, -1.0, 0.3, -7.7e-4, 1234.567, 3e-39, 1e-45, 70000.0, -2.5e36):
        d = np.float32(d)
        b = np.empty(32, np.float32)
        b[0] = d * np.float32(-8)
        steps = (np.arange(31) - 15) / 2.0 * np.float64(d)
        b[1:] = np.clip(steps, -abs(np.float64(b[0])), abs(np.float64(b[0]))).astype(np.float32)
        rows += [b, np.nextafter(b, np.float32(np.inf)), np.nextafter(b, np.float32(-np.inf))]
        rows[-2][0] = rows[-1][0] = b[0]
    rows.append(np.zeros(32, np.float32))
    for first, second in ((2.0, -2.0), (-2.0, 2.0)):
        b = np.linspace(-1, 1, 32).astype(np.float32)
        b[5], b[29] = first, second
        rows.append(b)
    for bad in (np.nan, np.inf, -np.inf):
        b = np.linspace(-1, 1, 32).astype(np.float32)
        b[17] = bad
        rows.append(b)
    x = np.stack(rows)
    got, want = store(x, np.arange(len(rows)), len(rows))
    assert np.array_equal(got, want)


@pytest.mark.parametrize("n,rows,cache", [(32, 1, 1), (1024, 1, 50), (1056, 37, 60), (128, 5000, 700)])
def test_read(n, rows, cache):
    r = np.random.default_rng([n, rows])
    row = n // 32 * 18 + 4
    raw = r.integers(0, 256, (cache, row)).astype(np.uint8)
    raw[:, 1:n // 32 * 18:18] &= 0xBF  # (finite scales)
    idx = r.integers(-1, cache + 1, rows).astype(np.int64)
    idx[0] = cache - 1
    if rows > 2:
        idx[2] = (1 << 32) + 1
    bs, bi, by = kc.Buffer.of(raw), kc.Buffer.of(idx), kc.Buffer(4 * rows * n + 64)
    by.upload(np.full(16, 9.0, np.float32), 4 * rows * n)
    kc.launch("get_rows_q4_0", kc.GetRowsQ40Args(bs.ptr, bi.ptr, by.ptr, n, rows, cache, row))
    got = by.download(np.float32)
    assert (got[rows * n:] == 9.0).all()
    values = unpack_q4(raw[:, :n // 32 * 18]).astype(np.float32)  # (15 bits: exact)
    want = np.where(((idx >= 0) & (idx < cache))[:, None], values[np.clip(idx, 0, cache - 1)], np.float32(0))
    assert np.array_equal(got[:rows * n].reshape(rows, n), want)
    for b in (bs, bi, by):
        b.free()


def plain_keep(w, n_keep, first, recent):
    T = w.shape[1]
    key = np.where(np.isnan(w), -np.inf, np.where(w == 0, 0.0, w))
    out = []
    for h in range(w.shape[0]):
        free = np.arange(first, T - recent)
        order = sorted(free, key=lambda i: (bool(np.isnan(w[h, i])), -key[h, i], i))[:n_keep - first - recent]
        out.append(np.sort(np.concatenate([np.arange(first), order, np.arange(T - recent, T)]).astype(np.int32)))
    return np.stack(out)


@pytest.mark.parametrize("heads,T,n_keep,first,recent", [(1, 1, 1, 0, 0), (3, 5, 5, 0, 0), (2, 64, 10, 0, 0), (2, 65, 33, 4, 7), (2, 1000, 999, 1, 1), (2, 1000, 1, 0, 0),
                                                         (3, 1025, 512, 4, 64), (1, 70000, 3000, 4, 256), (2, 300, 20, 4, 16), (2, 50, 0, 0, 0), (2, 40, 40, 20, 20)])
@pytest.mark.parametrize("kind", ["random", "ties", "special"])
def test_keep(heads, T, n_keep, first, recent, kind):
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
    got = bk.download(np.int32)
    want = np.full(heads * krow + 16, -7, np.int32)
    want[:heads * krow].reshape(heads, krow)[:, :n_keep] = plain_keep(w, n_keep, first, recent)
    assert np.array_equal(got, want)
    bw.free(), bk.free()


@pytest.mark.parametrize("heads,T,n,sizes", [(2, 50, 20, (256, 72, 4, 4)), (1, 1, 1, (2,)), (8, 300, 299, (128, 36)), (3, 4000, 1777, (6, 512, 144))])
def test_gather(heads, T, n, sizes):
    r = np.random.default_rng([T, n])
    keep = np.stack([np.sort(r.choice(T, n, replace=False)) for _ in range(heads)]).astype(np.int32)
    if n > 3:
        keep[0, 1], keep[0, 2] = -1, T  # left as they are
    bufs, planes, want = [], [], []
    for k, b in enumerate(sizes):
        # rows of all heads together, or heads apart; odd paddings
        srow, shead = (heads * b + 2, b) if k % 2 == 0 else (b, T * b + 6)
        drow, dhead = (b, n * b + 2) if k % 3 == 0 else (heads * b, b)
        src = r.integers(0, 256, (T - 1) * srow + (heads - 1) * shead + b).astype(np.uint8)
        dst = r.integers(0, 256, (n - 1) * drow + (heads - 1) * dhead + b + 32).astype(np.uint8)
        bs, bd = kc.Buffer.of(src), kc.Buffer.of(dst)
        out = dst.copy()
        for g in range(heads):
            for i in range(n):
                if 0 <= keep[g, i] < T:
                    at = keep[g, i] * srow + g * shead
                    out[i * drow + g * dhead:i * drow + g * dhead + b] = src[at:at + b]
        bufs.append((bs, bd))
        want.append(out)
        planes.append(kc.KvPlane(bs.ptr, bd.ptr, srow, shead, drow, dhead, b))
    bk = kc.Buffer.of(keep)
    kc.launch("kv_gather", kc.KvGatherArgs((kc.KvPlane * 4)(*planes), len(sizes), bk.ptr, heads, n, n, T))
    for (bs, bd), out in zip(bufs, want):
        assert np.array_equal(bd.download(np.uint8), out)
        bs.free(), bd.free()
    bk.free()
