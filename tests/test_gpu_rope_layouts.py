"""rope_ext on arrays that lie beside each other -- q, k and v of a token in one row with q turned in place, K and V in one cache row or one
head -- gives the bits that it gives on arrays of their own, and leaves the rest as it was. flash_pages_f16 reads such a cache."""
import numpy as np
import pytest

import kernelcore_amd as kc
from tests.serve import Out, Pages, up
from tests.test_gpu_rope_ext import run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def runtime():
    kc.init()
    yield
    kc.synchronize()


def at(flat, base, n, row, heads, head, D):
    """The values of n rows of heads in a flat array, by strides in values."""
    return flat[base + np.arange(n)[:, None, None] * row + np.arange(heads)[None, :, None] * head + np.arange(D)]


@pytest.mark.parametrize("inter", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("N", [1, 2, 37, 1300])
@pytest.mark.parametrize("H,K,D,n_rot", [(8, 2, 128, 128), (3, 1, 80, 36), (5, 5, 6, 2)])
@pytest.mark.parametrize("cache", ["row", "head", "outer"])
def test_beside(inter, N, H, K, D, n_rot, cache):
    print("rope_ext", inter, N, H, K, D, n_rot, cache, flush=True)
    r = np.random.default_rng([N, H, D])
    rows, T = N + 5, (H + 2 * K) * D + 3
    x = r.standard_normal(N * T).astype(np.float32)
    freqs, _ = kc.rope_freqs(n_rot, 1e4)
    small = dict(pos=up(r.integers(0, 100000, N), np.int32), freqs=up(freqs, np.float64), slots=up(r.permutation(rows)[:N], np.int64))
    p = {n: b.ptr for n, b in small.items()}
    sizes = dict(n_tokens=N, H=H, H_kv=K, D=D, n_rot=n_rot, interleaved=int(inter), cache_rows=rows, scale=1.25)
    q, k, v = (at(x, o * D, N, T, h, D, D) for o, h in ((0, H), (H, K), (H + K, K)))
    own = {n: up(a, np.float32) for n, a in dict(q=q, k=k, v=v).items()}
    qo, ko, vo = Out(q.size, np.float32), Out(rows * K * D, np.uint16, np.full(rows * K * D, 7)), Out(rows * K * D, np.uint16, np.full(rows * K * D, 7))
    kc.launch("rope_ext", kc.RopeExtArgs(**p, **{n: b.ptr for n, b in own.items()}, q_out=qo.ptr, k_cache=ko.ptr, v_cache=vo.ptr, q_tok=H * D, q_head=D, k_tok=K * D,
                                         k_head=D, v_tok=K * D, v_head=D, out_tok=H * D, out_head=D, kc_row=2 * K * D, kc_head=2 * D, vc_row=2 * K * D,
                                         vc_head=2 * D, **sizes))
    # in one buffer, and in one cache
    row, head, second = dict(row=(2 * K * D, D, K * D), head=(2 * K * D, 2 * D, D), outer=(2 * D, 2 * D * rows, D))[cache]
    before = np.arange(2 * K * D * rows, dtype=np.uint16) | 1
    xo, co = Out(x.size, np.float32, x), Out(before.size, np.uint16, before)
    kc.launch("rope_ext", kc.RopeExtArgs(**p, q=xo.ptr, k=xo.ptr + 4 * H * D, v=xo.ptr + 4 * (H + K) * D, q_out=xo.ptr, k_cache=co.ptr, v_cache=co.ptr + 2 * second, q_tok=T,
                                         q_head=D, k_tok=T, k_head=D, v_tok=T, v_head=D, out_tok=T, out_head=D, kc_row=2 * row, kc_head=2 * head, vc_row=2 * row,
                                         vc_head=2 * head, **sizes))
    kc.synchronize()
    want, want_cache = x.copy(), before.copy()
    where = at(np.arange(x.size), 0, N, T, H, D, D)
    want[where] = qo.get().reshape(N, H, D)
    assert np.array_equal(xo.get().view(np.uint32), want.view(np.uint32))
    live = np.zeros(rows, bool)
    live[small["slots"].download(np.int64)[:N]] = True
    for out, base in ((ko, 0), (vo, second)):
        where = at(np.arange(before.size), base, rows, row, K, head, D)
        want_cache[where[live]] = out.get().reshape(rows, K, D)[live]
    assert np.array_equal(co.get(), want_cache)
    for b in [*small.values(), *own.values()]:
        b.free()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("by", ["row", "head"])
def test_attention_of_a_shared_cache(D, by):
    """The bits of separate caches."""
    c = Pages(8, 2, D, [300, 77, 5], [20, 1, 5], 16, tree=True)
    want = c.attend(extra=0)[0]
    both = np.concatenate([c.k, c.v], 1) if by == "row" else np.stack([c.k, c.v], 2)
    b = c.upload()
    kv = up(both, np.float16)
    b.pop("k").free(), b.pop("v").free()
    head = 2 * D if by == "row" else 4 * D
    d = c.dims(k_row=8 * D, v_row=8 * D, k_head=head, v_head=head)
    part, out = Out(kc.flash_pages_part_bytes(d), np.uint8), Out(c.q.size, np.float32)
    kc.launch("flash_pages_f16", kc.FlashPagesArgs(**{n: x.ptr for n, x in b.items()}, k=kv.ptr, v=kv.ptr + (4 * D if by == "row" else 2 * D), out=out.ptr, part=part.ptr,
                                                   d=d, scale=c.scale))
    kc.synchronize()
    part.get()
    assert np.array_equal(out.get().reshape(c.q.shape), want)
    for x in [kv, *b.values()]:
        x.free()


@pytest.mark.parametrize("N", [8192, 10240, 10241, 18433, 30000])
@pytest.mark.parametrize("rows", [50, 20000])
def test_repeated_slots_of_many_tokens(N, rows):
    """The last token with a slot is stored, wherever the others with it are."""
    slots = np.random.default_rng(N).integers(-3, rows + 3, N)
    run(N, 1, 2, 8, 8, False, rows=rows, slots=slots)
    run(N, 2, 1, 6, 4, True, rows=rows, slots=slots, in_place=True, v=False)
