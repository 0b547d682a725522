"""What the cache operators refuse, on the CPU: the library over a stand-in for the HIP runtime (tests/hip_stub), so that each
call's arguments are checked and nothing runs. And the plain forms' own blocks."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np

import kernelcore_amd as kc
from tests.kvcache import pack_q4, unpack_q4

HERE = os.path.dirname(os.path.abspath(__file__))

CHILD = r"""
import ctypes as C, sys
stub = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
stub.stub_record.restype = C.c_char_p
import kernelcore_amd as kc
kc.init()
F32 = kc.Buffer(1 << 22).ptr
INF, NAN = float("inf"), float("nan")


def status(name, args):
    stub.stub_clear()
    r = kc.launch_status(name, args)
    if r != "Success":
        assert stub.stub_record() == b"", name  # refused before anything is launched
    return r


def checks(name, make, good, bad):
    assert status(name, make(**good)) == "Success", (name, kc.lib().kcGetLastErrorDetail())
    for change, want in bad:
        got = status(name, make(**dict(good, **change)))
        assert got == want, (name, change, got)


IV, IP = "InvalidValue", "InvalidPointer"
# ---- rows
def buf(n):
    return kc.Buffer(n).ptr

n, rows, cache = 128, 6, 20
good = dict(src=buf(4 * n * rows), idx=buf(8 * rows), dst=buf(72 * cache), n=n, rows=rows, src_row=n, dst_rows=cache, dst_row=72)
checks("set_rows_q4_0", lambda **k: kc.SetRowsQ40Args(**k), good,
       [(dict(n=0), IV), (dict(n=100), IV), (dict(rows=-1), IV), (dict(rows=1 << 20), IV), (dict(src_row=n - 1), IV), (dict(dst_rows=-1), IV),
        (dict(dst_row=70), IV), (dict(dst_row=73), IV), (dict(dst_row=1 << 62), IV), (dict(src=None), IP), (dict(idx=None), IP), (dict(dst=None), IP),
        (dict(rows=7), IP), (dict(dst_rows=21), IP), (dict(src=good["src"] + 2), IV), (dict(dst=good["dst"] + 1), IV), (dict(idx=good["idx"] + 2), IV)])
good = dict(src=buf(72 * cache), idx=buf(8 * rows), y=buf(4 * n * rows), n=n, rows=rows, src_rows=cache, src_row=72)
checks("get_rows_q4_0", lambda **k: kc.GetRowsQ40Args(**k), good,
       [(dict(n=0), IV), (dict(n=33), IV), (dict(rows=-1), IV), (dict(src_rows=-1), IV), (dict(src_row=71), IV), (dict(src_row=70), IV), (dict(src=None), IP),
        (dict(y=None), IP), (dict(rows=7), IP), (dict(src_rows=21), IP), (dict(src=good["src"] + 1), IV), (dict(y=good["y"] + 1), IV)])

# ---- attention
DIMS = dict(H=8, H_kv=2, D=128, N=3, T=700, q_tok=1024, q_head=128, m_row=350, key_row=700, pos0=697, causal=1, prefix=0)
for q4 in (False, True):
    hb = 72 if q4 else 256
    dims = dict(DIMS, k_row=2 * hb, k_head=hb, v_row=2 * hb, v_head=hb)
    part = kc.flash_ext_part_bytes(kc.FlashExtDims(**dims))
    assert part > 0
    common = dict(q=buf(4 * 3 * 1024), k=buf(2 * hb * 700), mask=buf(3 * 700 * 2), qpos=buf(12), kpos=buf(4 * 1400), qdoc=buf(12), kdoc=buf(4 * 1400),
                  slopes=buf(32), scale=0.1, softcap=0.0)
    extra = dict(v=buf(2 * hb * 700), out=buf(4 * 3 * 1024), lse=buf(4 * 24), part=buf(part))
    wextra = dict(lse=extra["lse"], w_in=buf(4 * 1400), w=buf(4 * 1400), w_row=700, decay=0.9)

    def build(cls):
        def make(**k):
            d = {n: k.pop(n) for n in list(dims)}
            return cls(d=kc.FlashExtDims(**d), **k)
        return make

    shared = [(dict(H=0), IV), (dict(H=7), IV), (dict(H_kv=0), IV), (dict(D=96), IV), (dict(D=0), IV), (dict(N=-1), IV), (dict(T=-1), IV), (dict(T=2**31 - 1), IV), (dict(T=2**31 - 1024), IV),
              (dict(q_tok=-1), IV), (dict(q_head=-4), IV), (dict(k_row=-2), IV), (dict(key_row=-1), IV), (dict(key_row=699), IV), (dict(causal=2), IV),
              (dict(prefix=-1), IV), (dict(pos0=-1), IV), (dict(pos0=2**31 - 3), IV), (dict(N=1 << 24), IV), (dict(k_row=2 * hb + 1), IV), (dict(k_head=hb + 1), IV),
              (dict(k_row=1 << 61), IV), (dict(scale=NAN), IV), (dict(scale=INF), IV), (dict(softcap=-1.0), IV), (dict(softcap=NAN), IV), (dict(softcap=INF), IV),
              (dict(qdoc=None), IV), (dict(kdoc=None), IV), (dict(m_row=349), IV), (dict(q=None), IP), (dict(k=None), IP), (dict(N=4), IP),
              (dict(T=701, key_row=701, m_row=351), IP), (dict(k=common["k"] + 1), IV), (dict(q=common["q"] + 2), IV), (dict(mask=common["mask"] + 2), IV),
              (dict(kpos=common["kpos"] + 4), IP), (dict(slopes=common["slopes"] + 4), IP), (dict(qpos=common["qpos"] + 4), IP), (dict(q_tok=1025), IP)]
    if not q4:
        shared += [(dict(k_row=2 * hb + 2), IV), (dict(k=common["k"] + 2), IV)]
    t = "_q4_0" if q4 else "_f16"
    checks("flash_ext" + t, build(kc.FlashExtArgs), dict(dims, **common, **extra), shared +
           [(dict(v_row=-2), IV), (dict(v_row=2 * hb + 1), IV), (dict(v=None), IP), (dict(out=None), IP), (dict(part=None), IP), (dict(part=extra["part"] + 4), IP),
            (dict(lse=extra["lse"] + 4), IP), (dict(out=extra["out"] + 2), IV)])
    checks("attn_weights" + t, build(kc.AttnWeightsArgs), dict(dims, **common, **wextra), shared +
           [(dict(w_row=699), IV), (dict(decay=NAN), IV), (dict(lse=None), IP), (dict(w=None), IP), (dict(w_in=wextra["w_in"] + 4), IP), (dict(w=wextra["w"] + 2), IV)])
    # what may be absent
    for gone in (("mask",), ("qpos",), ("kpos",), ("qdoc", "kdoc"), ("slopes",), ("lse",)):
        a = dict(dims, **common, **extra)
        a.update({g: None for g in gone})
        assert status("flash_ext" + t, build(kc.FlashExtArgs)(**a)) == "Success", gone
    assert status("flash_ext" + t, build(kc.FlashExtArgs)(**dict(dict(dims, **common, **extra), N=0))) == "Success"
    assert status("flash_ext" + t, build(kc.FlashExtArgs)(**dict(dict(dims, **common, **extra), T=0, part=None))) == "Success"
n = C.c_size_t()
assert kc.lib().kcFlashExtPartBytes(None, C.byref(n)) == kc.ERR["InvalidValue"]
assert kc.lib().kcFlashExtPartBytes(C.byref(kc.FlashExtDims(**dict(dims, D=32))), C.byref(n)) == kc.ERR["InvalidValue"]

# ---- positions and rows to keep
good = dict(w=buf(4 * 2 * 100), keep=buf(4 * 2 * 40), heads=2, T=100, w_row=100, n_keep=40, keep_row=40, first=4, recent=8)
checks("kv_keep", lambda **k: kc.KvKeepArgs(**k), good,
       [(dict(heads=0), IV), (dict(T=-1), IV), (dict(w_row=99), IV), (dict(first=-1), IV), (dict(recent=-1), IV), (dict(n_keep=101, keep_row=101), IV), (dict(first=33), IV),
        (dict(keep_row=39), IV), (dict(w=None), IP), (dict(keep=None), IP), (dict(heads=3), IP), (dict(T=101, w_row=101), IP), (dict(w=good["w"] + 2), IV)])
src, dst, keep = buf(100 * 512), buf(40 * 512), buf(4 * 80)


def gather(**k):
    p = dict(src=src, dst=dst, src_row=512, src_head=256, dst_row=512, dst_head=256, bytes=256)
    p.update({n: k.pop(n) for n in list(k) if n in p})
    args = dict(dict(n_planes=1, keep=keep, heads=2, n_keep=40, keep_row=40, T=100), **k)
    return kc.KvGatherArgs(planes=(kc.KvPlane * 4)(*[kc.KvPlane(**p)] * 4), **args)


checks("kv_gather", gather, {},
       [(dict(n_planes=0), IV), (dict(n_planes=5), IV), (dict(heads=0), IV), (dict(n_keep=-1), IV), (dict(T=-1), IV), (dict(keep_row=39), IV), (dict(bytes=0), IV),
        (dict(bytes=255), IV), (dict(src_row=254), IV), (dict(dst_row=254), IV), (dict(src_head=-256), IV), (dict(dst_head=254), IV), (dict(src_row=511), IV),
        (dict(keep=None), IP), (dict(src=None), IP), (dict(dst=None), IP), (dict(T=101), IP), (dict(n_keep=41, keep_row=41), IP), (dict(src=src + 1), IV),
        (dict(dst=src), IV), (dict(dst=src + 512), IV), (dict(src_row=1 << 62), IV)])
print("done")
"""


def test_refusals(tmp_path):
    stub = str(tmp_path / "hip_stub.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", os.path.join(HERE, "hip_stub", "hip_stub.cpp"), "-o", stub],
                   check=True)
    r = subprocess.run([sys.executable, "-c", CHILD, stub], capture_output=True, text=True, cwd=os.path.dirname(HERE), timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["done"], r.stdout + r.stderr


def test_plain_blocks():
    """Nearest codes: a value is off by at most half a step of its block and the scale's own rounding."""
    x = np.random.default_rng(0).standard_normal((50, 96)).astype(np.float32)
    y = unpack_q4(pack_q4(x))
    top = np.abs(x.reshape(50, 3, 32)).max(-1, keepdims=True)
    err = np.abs(x.reshape(50, 3, 32) - y.reshape(50, 3, 32))
    # half a step (top / 16), a whole one for a value beyond the last code on the other side, and 2^-11 of the value
    assert (err <= top / 8 + top * 2.0 ** -11).all()
    inner = x.reshape(50, 3, 32) * np.sign(np.take_along_axis(x.reshape(50, 3, 32), np.abs(x.reshape(50, 3, 32)).argmax(-1)[..., None], -1)) >= -top * 7 / 8
    assert (err[inner] <= np.broadcast_to(top / 16 + top * 2.0 ** -11, err.shape)[inner]).all()


STRUCTS = ["SetRowsQ40Args", "GetRowsQ40Args", "FlashExtDims", "FlashExtArgs", "AttnWeightsArgs", "KvKeepArgs", "KvPlane", "KvGatherArgs"]


def test_struct_layouts(tmp_path):
    """The ctypes structures against what gcc makes of the C header."""
    lines = ["#include <stdio.h>", "#include <stddef.h>", "#include <kernelcore/llm_kernels.h>", "int main(void) {"]
    for s in STRUCTS:
        lines.append(f'printf("{s} %zu\\n", sizeof(kc{s}));')
        lines += [f'printf("{s}.{f} %zu\\n", offsetof(kc{s}, {f}));' for f, _ in getattr(kc, s)._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0;", "}"]))
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-std=c11", f"-I{kc.ROOT}/include", str(tmp_path / "layout.c"), "-o", exe], check=True)
    want = dict(line.split() for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines())
    for s in STRUCTS:
        cls = getattr(kc, s)
        assert int(want[s]) == C.sizeof(cls), s
        for f, _ in cls._fields_:
            assert int(want[f"{s}.{f}"]) == getattr(cls, f).offset, f"{s}.{f}"
