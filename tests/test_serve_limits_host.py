"""Which memory layouts and sizes the operators of a step over a paged cache accept, on the CPU (the library over tests/hip_stub, as in
test_serve_host.py)."""
import os
import subprocess
import sys

import numpy as np
import pytest

import kernelcore_amd as kc
from tests.test_serve_host import CHILD, HERE

PRELUDE = CHILD[:CHILD.index("# ---- kv_pages")]


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    path = str(tmp_path_factory.mktemp("stub") / "hip_stub.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", os.path.join(HERE, "hip_stub", "hip_stub.cpp"), "-o", path],
                   check=True)
    return path


def run(stub, code):
    r = subprocess.run([sys.executable, "-c", PRELUDE + code + '\nprint("done")\n', stub], capture_output=True, text=True, cwd=os.path.dirname(HERE), timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["done"], r.stdout + r.stderr


def test_rope_layouts(stub):
    """Arrays that lie beside each other are accepted wherever they share no value, and refused where they share one."""
    run(stub, r"""
import numpy as np
r = np.random.default_rng(0)
N, H, K, D, ROWS = 5, 4, 2, 64, 7
T = (H + 2 * K) * D
qkv, small, cache = buf(4 * N * T), dict(pos=buf(4 * N), freqs=buf(8 * 16), slots=buf(8 * N)), buf(2 * ROWS * 2 * K * D)
make = lambda **k: kc.RopeExtArgs(**k)  # noqa: E731
good = dict(small, q=qkv, k=qkv + 4 * H * D, v=qkv + 4 * (H + K) * D, q_out=qkv, k_cache=cache, v_cache=cache + 2 * K * D, n_tokens=N, H=H, H_kv=K, D=D, n_rot=32,
            q_tok=T, q_head=D, k_tok=T, k_head=D, v_tok=T, v_head=D, out_tok=T, out_head=D, cache_rows=ROWS, kc_row=4 * K * D, kc_head=2 * D, vc_row=4 * K * D,
            vc_head=2 * D, scale=1.0)
checks("rope_ext", make, good,
       [(dict(kc_head=4 * D, vc_head=4 * D, v_cache=cache + 2 * D), OK),  # K and V of a head side by side
        (dict(kc_row=2 * D, vc_row=2 * D, kc_head=4 * D * ROWS, vc_head=4 * D * ROWS, v_cache=cache + 2 * D * ROWS), OK),  # heads outermost, K's rows then V's
        (dict(kc_row=4 * D, vc_row=4 * D, kc_head=4 * D * ROWS, vc_head=4 * D * ROWS, v_cache=cache + 2 * D), OK),  # and side by side in each row
        (dict(q_out=qkv + 4 * D * H, k=qkv, k_head=D), IV), (dict(k=qkv + 4 * (H * D - 1)), IV), (dict(v=qkv), IV), (dict(v_cache=cache + 2 * K * D - 2), IV),
        (dict(v_cache=cache + 2 * D), IV), (dict(kc_head=4 * D, vc_head=4 * D, v_cache=cache + 2 * D - 2), IV), (dict(out_tok=T - D, n_tokens=4), IV)])
# Layouts of two arrays at random: refused if they share a value, accepted if they do not and lie beside each other at a common distance.
n, h, d, base = 3, 2, 2, buf(4096)
seen = {OK: 0, IV: 0}
for _ in range(8000):
    step = lambda: int(r.choice([4, 6, 8, 12, 16, 24, 32, 48]))  # noqa: E731
    k = (2 * int(r.integers(0, 60)), step(), step())  # offset, bytes between rows, between heads
    v = (2 * int(r.integers(0, 60)), *(k[1:] if r.random() < 0.6 else (step(), step())))
    if not all((head >= 2 * d and row >= head + 2 * d) or (row >= 2 * d and head >= 2 * row + 2 * d) for _, row, head in (k, v)):
        continue  # rows and heads through each other are refused anyway
    values = [{at + i * row + j * head + 2 * e for i in range(n) for j in range(h) for e in range(d)} for at, row, head in (k, v)]
    got = status("rope_ext", make(**dict(small, k=qkv, v=qkv, k_cache=base + k[0], v_cache=base + v[0], n_tokens=2, H_kv=h, D=d, n_rot=2, k_tok=4, k_head=2, v_tok=4,
                                         v_head=2, cache_rows=n, kc_row=k[1], kc_head=k[2], vc_row=v[1], vc_head=v[2], scale=1.0)))
    seen[got] += 1
    if values[0] & values[1]:
        assert got == IV, (k, v)
    elif k[1:] == v[1:]:
        size = {k[1]: (h - 1) * k[2] + 2 * d, k[2]: (n - 1) * k[1] + 2 * d}
        if any(size[x] <= (v[0] - k[0]) % x <= x - size[x] for x in size):
            assert got == OK, (k, v)
assert min(seen.values()) > 300, seen
""")


@pytest.mark.parametrize("N", [1, 8192, 10240, 10241, 40000, (1 << 20) + 1])
def test_rope_launches(stub, N):
    """A launch's search for repeated slots is bounded: many tokens take several launches, each with a part of them."""
    run(stub, f"N = {N}" + r"""
b = {n: buf(8 * N) for n in ("q", "k", "v", "pos", "freqs", "slots", "q_out", "k_cache", "v_cache")}
args = dict(b, n_tokens=N, H=1, H_kv=1, D=2, n_rot=2, q_tok=2, q_head=2, k_tok=2, k_head=2, v_tok=2, v_head=2, out_tok=2, out_head=2, cache_rows=N, kc_row=4, kc_head=4,
            vc_row=4, vc_head=4, scale=1.0)
for change in ({}, dict(q=None, q_out=None), dict(k=None, k_cache=None, v=None, v_cache=None, slots=None)):
    assert status("rope_ext", kc.RopeExtArgs(**dict(args, **change))) == OK
    grids = [int(x.split()[-4]) for x in stub.stub_record().decode().splitlines()]
    # (a workgroup has at most 16 tokens)
    stores = "k" not in change
    assert len(grids) == (max(1, (N + 6143) // 8192) if stores else -(-N // (1 << 20))) and max(grids) <= (2 * 10240 if stores else 1 << 20), grids
    assert sum(grids) >= N // 16
stub.stub_clear()
assert kc.launch_status("rope_ext", kc.RopeExtArgs(**dict(args, q=None, q_out=None, k=None, k_cache=None, v=None, v_cache=None, slots=None))) == OK
assert stub.stub_record() == b""  # neither q nor k: nothing to do
""")


@pytest.mark.parametrize("N", [0, 1, 1 << 18, (1 << 18) + 1, 1000000])
def test_tree_launches(stub, N):
    """A launch's walks up the trees are bounded by its tokens; without trees there is one launch."""
    run(stub, f"N = {N}" + r"""
b = {n: buf(max(16, 8 * N)) for n in ("have", "add", "free", "table", "start", "len", "slots", "pos", "used", "parent", "tree")}
for tree in (True, False):
    a = dict(b) if tree else dict(b, parent=None, tree=None)
    assert status("kv_pages", kc.KvPagesArgs(**a, seqs=2, n_tokens=N, n_free=1, page=16, max_pages=1, table_row=1, tree_words=2 if tree else 0)) == OK
    grids = [int(x.split()[-4]) for x in stub.stub_record().decode().splitlines()]
    assert sum(grids) == max(1, -(-N // 256)) and len(grids) == (max(1, -(-N // (1 << 18))) if tree else 1), grids
""")


def test_pages_sizes(stub):
    """Each workgroup of tokens sums over the sequences before them: both are bounded."""
    run(stub, r"""
M = 1 << 24
b = {n: buf(8 * M + 16) for n in ("have", "add", "free", "table", "start", "len", "slots", "pos", "used")}
checks("kv_pages", lambda **k: kc.KvPagesArgs(**k), dict(b, seqs=M, n_tokens=M, n_free=1, page=16, max_pages=1, table_row=1),
       [(dict(seqs=M + 1), IV), (dict(n_tokens=M + 1), IV), (dict(seqs=M + 1, n_tokens=0), IV), (dict(seqs=0, n_tokens=M + 1), IV), (dict(seqs=1), OK), (dict(n_tokens=1), OK)])
""")


def test_attention_sizes(stub):
    """A launch has fewer than 2^32 threads."""
    run(stub, r"""
d = dict(H=2, H_kv=1, D=64, N=8, seqs=(1 << 24) - 2, page=16, max_pages=1, n_pages=1, tree_words=0, q_tok=128, q_head=64, table_row=1, k_row=128, k_head=128, v_row=128, v_head=128)
b = C.c_size_t()
size = lambda **k: kc.lib().kcFlashPagesPartBytes(C.byref(kc.FlashPagesDims(**dict(d, **k))), C.byref(b))  # noqa: E731
assert size() == kc.ERR[OK] and size(N=7, seqs=d["seqs"] + 1) == kc.ERR[OK]
assert size(N=16) == size(N=7, seqs=d["seqs"] + 2) == size(seqs=d["seqs"] + 1) == size(N=0, seqs=1 << 24) == kc.ERR[IV]
size()
n = 4 * d["seqs"] + 4
a = {x: buf(n) for x in ("table", "start", "len")}
args = dict(a, q=buf(4096 * 2), k=buf(4096), v=buf(4096), out=buf(4096 * 2), part=buf(b.value), scale=0.1)
stub.stub_clear()
assert kc.launch_status("flash_pages_f16", kc.FlashPagesArgs(d=kc.FlashPagesDims(**d), **args)) == OK, kc.lib().kcGetLastErrorDetail()
for x in stub.stub_record().decode().splitlines():
    assert int(x.split()[-4]) * int(x.split()[-1]) < 1 << 32, x
""")


def test_sample_workspace(stub):
    """A workspace made for some rows is enough for fewer of them."""
    run(stub, r"""
for V in (1, 1000, 65536, 65537, 128256, 151936, 1 << 20):
    need = [kc.sample_rows_part_bytes(R, V) for R in range(200)]
    assert need == sorted(need) and need[0] == 0, V
R, V = 40, 151936
a = dict(logits=buf(4 * R * V), u=buf(4 * R), tokens=buf(4 * R), part=buf(kc.sample_rows_part_bytes(R, V)), row=V, n_vocab=V)
for rows in range(R + 1):
    assert status("sample_rows", kc.SampleRowsArgs(**a, rows=rows)) == OK, rows
    for x in stub.stub_record().decode().splitlines()[:1]:
        assert int(x.split()[-4]) * int(x.split()[-3]) * 20496 <= kc.sample_rows_part_bytes(rows, V)  # 2048 sums, 1024 maxima and three numbers a piece
""")


@pytest.mark.parametrize("bad", [0.0, -0.0, -1.0, float("nan"), float("inf"), float("-inf")])
def test_frequency_factors(bad):
    """A factor that would make a frequency infinite, NaN, 0 or turn it round is refused."""
    for at in (0, 5, 31):
        ff = np.ones(32, np.float32)
        assert np.isfinite(kc.rope_freqs(64, 1e4, ff=ff)[0]).all()
        ff[at] = bad
        with pytest.raises(kc.KcError, match="InvalidValue"):
            kc.rope_freqs(64, 1e4, ff=ff)
