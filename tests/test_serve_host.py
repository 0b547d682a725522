"""What the operators of a step over a paged cache refuse, on the CPU: the library over a stand-in for the HIP runtime (tests/hip_stub), so that
each call's arguments are checked and nothing runs. And kcRopeFreqs, a host function, against its formula."""
import ctypes as C
import math
import os
import subprocess
import sys

import numpy as np
import pytest

import kernelcore_amd as kc
from tests.serve import plain_pages, plain_sample

HERE = os.path.dirname(os.path.abspath(__file__))

CHILD = r"""
import ctypes as C, sys
stub = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
stub.stub_record.restype = C.c_char_p
import kernelcore_amd as kc
kc.init()
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
        assert got == want, (name, change, got, kc.lib().kcGetLastErrorDetail())


IV, IP, OK = "InvalidValue", "InvalidPointer", "Success"


def buf(n):
    return kc.Buffer(n).ptr


# ---- kv_pages
S, N = 5, 40
good = dict(have=buf(4 * S), add=buf(4 * S), free=buf(4 * 30), parent=buf(4 * N), table=buf(4 * (9 * 4 + 7)), start=buf(4 * S + 4), len=buf(4 * S), slots=buf(8 * N),
            pos=buf(4 * N), used=buf(4), tree=buf(8 * N), seqs=S, n_tokens=N, n_free=30, page=16, max_pages=7, table_row=9, tree_words=2)
checks("kv_pages", lambda **k: kc.KvPagesArgs(**k), good,
       [(dict(seqs=-1), IV), (dict(n_tokens=-1), IV), (dict(n_free=-1), IV), (dict(page=0), IV), (dict(page=8), IV), (dict(page=48), IV), (dict(page=131072), IV),
        (dict(max_pages=-1), IV), (dict(max_pages=10), IV), (dict(tree_words=0), IV), (dict(tree_words=65), IV), (dict(parent=None), IV), (dict(tree=None), IV),
        (dict(parent=None, tree=None), IV), (dict(parent=None, tree=None, tree_words=0), OK), (dict(pos=None), OK), (dict(seqs=0), OK), (dict(n_tokens=0), OK),
        (dict(n_free=0, free=None), OK), (dict(max_pages=0), OK), (dict(n_tokens=2**31 - 1), IV), (dict(seqs=2**31 - 1), IV), (dict(have=None), IP), (dict(add=None), IP),
        (dict(free=None), IP), (dict(table=None), IP), (dict(start=None), IP), (dict(len=None), IP), (dict(slots=None), IP), (dict(used=None), IP), (dict(seqs=6), IP),
        (dict(n_tokens=41), IP), (dict(n_free=31), IP), (dict(max_pages=8), IP), (dict(table_row=10), IP), (dict(tree_words=3), IP), (dict(have=good["have"] + 2), IV),
        (dict(slots=good["slots"] + 4), IV), (dict(len=good["have"]), IV), (dict(pos=good["parent"]), IV), (dict(start=good["table"]), IV), (dict(used=good["len"] + 8), IV),
        (dict(pos=good["tree"] + 4 * N), IV), (dict(tree=good["tree"] + 4), IP)])

# ---- rope_ext
n, H, K, D = 6, 4, 2, 64
good = dict(q=buf(4 * n * H * D), k=buf(4 * n * K * D), v=buf(4 * 20 * K * D), pos=buf(4 * n), freqs=buf(8 * 16), slots=buf(8 * n), q_out=buf(4 * n * H * D),
            k_cache=buf(20 * K * D * 2), v_cache=buf(20 * K * D * 2), n_tokens=n, H=H, H_kv=K, D=D, n_rot=32, interleaved=0, q_tok=H * D, q_head=D, k_tok=K * D, k_head=D,
            v_tok=K * D, v_head=D, out_tok=H * D, out_head=D, cache_rows=20, kc_row=2 * K * D, kc_head=2 * D, vc_row=2 * K * D, vc_head=2 * D, scale=1.0)
checks("rope_ext", lambda **k: kc.RopeExtArgs(**k), good,
       [(dict(n_tokens=-1), IV), (dict(n_tokens=1 << 30), IV), (dict(D=0), IV), (dict(D=63), IV), (dict(D=1026), IV), (dict(n_rot=0), IV), (dict(n_rot=31), IV),
        (dict(n_rot=66), IV), (dict(interleaved=2), IV), (dict(scale=NAN), IV), (dict(scale=INF), IV), (dict(q=None), IV), (dict(q_out=None), IV), (dict(k=None), IV),
        (dict(k_cache=None), IV), (dict(v=None), IV), (dict(v_cache=None), IV), (dict(k=None, k_cache=None), IV), (dict(q=None, q_out=None), OK),
        (dict(v=None, v_cache=None), OK), (dict(k=None, k_cache=None, v=None, v_cache=None, slots=None), OK), (dict(n_tokens=0), OK), (dict(q_out=good["q"]), OK),
        (dict(q_out=good["q"], n_tokens=1, out_tok=0), IV), (dict(q_out=good["q"] + 4), IP), (dict(q_out=good["k"], n_tokens=3), IV), (dict(q_out=good["q"], out_tok=H * D + 2, n_tokens=5), IV),
        (dict(H=0), IV), (dict(H_kv=0), IV), (dict(H=70000), IV), (dict(cache_rows=-1), IV), (dict(q_tok=-1), IV), (dict(q_head=-1), IV), (dict(k_tok=-4), IV),
        (dict(out_tok=H * D - 1), IV), (dict(out_head=D - 1), IV), (dict(kc_row=2 * K * D - 2), IV), (dict(kc_head=2 * D - 2), IV), (dict(kc_head=2 * D + 1), IV),
        (dict(vc_row=2 * K * D + 1), IV), (dict(kc_row=-2), IV), (dict(kc_row=1 << 62), IV), (dict(k_cache=good["k_cache"] + 1), IV), (dict(v_cache=good["k_cache"]), IV),
        (dict(v_cache=good["v"]), IV), (dict(pos=None), IP), (dict(freqs=None), IP), (dict(slots=None), IP), (dict(n_rot=34), IP), (dict(n_tokens=7), IP),
        (dict(cache_rows=21), IP), (dict(pos=good["pos"] + 2), IV), (dict(freqs=good["freqs"] + 4), IV), (dict(slots=good["slots"] + 4), IV), (dict(q=good["q"] + 2), IV),
        (dict(kc_row=2 * D, kc_head=40 * D), OK), (dict(kc_row=2 * D, kc_head=40 * D - 2), IV), (dict(q_tok=0, q_head=0), OK), (dict(out_tok=0), IV)])

# ---- flash_pages_f16
dims = dict(H=8, H_kv=2, D=128, N=12, seqs=3, page=32, max_pages=5, n_pages=9, tree_words=2, q_tok=1024, q_head=128, table_row=6, k_row=512, k_head=256, v_row=512, v_head=256)
part = kc.flash_pages_part_bytes(kc.FlashPagesDims(**dims))
assert part > 0
good = dict(dims, q=buf(4 * 12 * 1024), k=buf(9 * 32 * 512), v=buf(9 * 32 * 512), table=buf(4 * 17), start=buf(16), len=buf(12), tree=buf(8 * 12), out=buf(4 * 12 * 1024),
            lse=buf(4 * 96), part=buf(part), scale=0.1)


def make(**k):
    d = {x: k.pop(x) for x in dims}
    return kc.FlashPagesArgs(d=kc.FlashPagesDims(**d), **k)


checks("flash_pages_f16", make, good,
       [(dict(H=0), IV), (dict(H=7), IV), (dict(H_kv=0), IV), (dict(D=96), IV), (dict(D=0), IV), (dict(N=-1), IV), (dict(seqs=-1), IV), (dict(page=8), IV), (dict(page=33), IV),
        (dict(max_pages=-1), IV), (dict(max_pages=7), IV), (dict(n_pages=-1), IV), (dict(n_pages=1 << 26), IV), (dict(n_pages=(1 << 26) - 1), IP), (dict(tree_words=0), IV), (dict(tree_words=65), IV), (dict(tree=None), IV),
        (dict(tree=None, tree_words=0), OK), (dict(lse=None), OK), (dict(N=0), OK), (dict(seqs=0), OK), (dict(n_pages=0), OK), (dict(max_pages=0), OK),
        (dict(page=65536, max_pages=32768, table_row=32768), IV), (dict(q_tok=-1), IV), (dict(q_head=-4), IV), (dict(k_row=-16), IV), (dict(k_row=520), IV), (dict(k_head=250), IV),
        (dict(v_row=528, v_head=8), IV), (dict(k_row=1 << 61), IV), (dict(k_row=1 << 27), IV), (dict(scale=NAN), IV), (dict(scale=INF), IV), (dict(q=None), IP), (dict(k=None), IP),
        (dict(v=None), IP), (dict(table=None), IP), (dict(start=None), IP), (dict(len=None), IP), (dict(out=None), IP), (dict(part=None), IP), (dict(N=13), IP), (dict(seqs=4), IP),
        (dict(n_pages=10), IP), (dict(max_pages=6), IP), (dict(tree_words=3), IP), (dict(k=good["k"] + 8), IV), (dict(part=good["part"] + 4), IV), (dict(part=good["part"] + 16), IP),
        (dict(q=good["q"] + 2), IV), (dict(out=good["out"] + 1), IV), (dict(lse=good["lse"] + 4), IP), (dict(start=good["start"] + 4), IP), (dict(len=good["len"] + 1), IV),
        (dict(N=1 << 22), IV), (dict(seqs=1 << 24), IV), (dict(out=good["q"]), IV), (dict(lse=good["out"]), IV), (dict(lse=good["tree"] + 4, N=0), OK),
        (dict(out=good["k"]), IV), (dict(lse=good["len"], N=1, H=2, q_head=0), IV), (dict(q=good["part"]), IV), (dict(table=good["part"]), IV)])
b = C.c_size_t()
assert kc.lib().kcFlashPagesPartBytes(None, C.byref(b)) == kc.ERR["InvalidValue"]
assert kc.lib().kcFlashPagesPartBytes(C.byref(kc.FlashPagesDims(**dims)), None) == kc.ERR["InvalidValue"]
assert kc.lib().kcFlashPagesPartBytes(C.byref(kc.FlashPagesDims(**dict(dims, page=17))), C.byref(b)) == kc.ERR["InvalidValue"]

# ---- sample_rows
R, V = 3, 1000
part = kc.sample_rows_part_bytes(R, V)
good = dict(logits=buf(4 * (2 * 1010 + V)), u=buf(12), temperature=buf(12), top_k=buf(12), top_p=buf(12), min_p=buf(12), tokens=buf(12), probs=buf(12), part=buf(part), row=1010,
            rows=R, n_vocab=V)
checks("sample_rows", lambda **k: kc.SampleRowsArgs(**k), good,
       [(dict(rows=-1), IV), (dict(rows=65536), IV), (dict(n_vocab=0), IV), (dict(n_vocab=(1 << 20) + 1), IV), (dict(row=-1), IV), (dict(row=1 << 62), IV), (dict(rows=0), OK),
        (dict(temperature=None), OK), (dict(top_k=None), OK), (dict(top_p=None), OK), (dict(min_p=None), OK), (dict(probs=None), OK), (dict(row=0), OK), (dict(logits=None), IP),
        (dict(u=None), IP), (dict(tokens=None), IP), (dict(part=None), IP), (dict(rows=4), IP), (dict(row=1011), IP), (dict(n_vocab=1001), IP), (dict(part=good["part"] + 16), IP),
        (dict(part=good["part"] + 8), IV), (dict(u=good["u"] + 2), IV), (dict(logits=good["logits"] + 1), IV), (dict(tokens=good["tokens"] + 4), IP), (dict(top_k=good["top_k"] + 4), IP),
        (dict(tokens=good["top_k"]), IV), (dict(probs=good["u"]), IV), (dict(probs=good["tokens"]), IV), (dict(part=good["logits"], rows=0), OK)])
for args in ((-1, 10), (70000, 10), (1, 0), (1, (1 << 20) + 1)):
    assert kc.lib().kcSampleRowsPartBytes(*args, C.byref(b)) == kc.ERR["InvalidValue"], args
assert kc.lib().kcSampleRowsPartBytes(1, 1, None) == kc.ERR["InvalidValue"]
print("done")
"""


def test_refusals(tmp_path):
    stub = str(tmp_path / "hip_stub.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", os.path.join(HERE, "hip_stub", "hip_stub.cpp"), "-o", stub],
                   check=True)
    r = subprocess.run([sys.executable, "-c", CHILD, stub], capture_output=True, text=True, cwd=os.path.dirname(HERE), timeout=300)
    assert r.returncode == 0 and r.stdout.split() == ["done"], r.stdout + r.stderr


STRUCTS = ["KvPagesArgs", "RopeScaling", "RopeExtArgs", "FlashPagesDims", "FlashPagesArgs", "SampleRowsArgs"]


def test_struct_layouts_match_the_c_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", "#include <kernelcore/llm_kernels.h>", "int main(void) {"]
    for s in STRUCTS:
        lines.append(f'printf("{s} %zu\\n", sizeof(kc{s}));')
        lines += [f'printf("{s}.{f} %zu\\n", offsetof(kc{s}, {f}));' for f, _ in getattr(kc, s)._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", f"-I{kc.ROOT}/include", str(src), "-o", str(exe)], check=True)
    want = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True).stdout.splitlines())
    for s in STRUCTS:
        assert int(want[s]) == C.sizeof(getattr(kc, s)), s
        for f, _ in getattr(kc, s)._fields_:
            assert int(want[f"{s}.{f}"]) == getattr(getattr(kc, s), f).offset, f"{s}.{f}"


# ---- kcRopeFreqs

@pytest.mark.parametrize("n_rot,base", [(2, 1e4), (64, 1e4), (128, 5e5), (1024, 1e6), (10, 1.5)])
@pytest.mark.parametrize("factor", [1.0, 4.0, 0.5])
def test_freqs_linear(n_rot, base, factor):
    ff = np.random.default_rng(0).uniform(1, 8, n_rot // 2).astype(np.float32)
    i = np.arange(n_rot // 2)
    for f in (None, ff):
        got, scale = kc.rope_freqs(n_rot, base, factor, ff=f)
        want = np.longdouble(np.float32(base)) ** (-2 * np.longdouble(1) * i / n_rot) / factor / (2 * np.pi) / (1 if f is None else f.astype(np.longdouble))
        # (a power of some 2^-53, a few more roundings, 2 pi in 64 bits)
        assert (np.abs(got - want) <= want * 2.0 ** -49).all() and scale == 1.0


@pytest.mark.parametrize("n_rot,base,factor,ctx", [(128, 1e6, 4.0, 32768), (64, 1e4, 32.0, 4096), (128, 5e5, 8.0, 8192), (32, 1e4, 2.0, 100)])
def test_freqs_yarn(n_rot, base, factor, ctx):
    got, scale = kc.rope_freqs(n_rot, base, factor, yarn_ctx=ctx)
    i = np.arange(n_rot // 2)
    plain = base ** (-2.0 * i / n_rot) / (2 * np.pi)
    turns = plain * ctx
    # pairs that turn more than 32 times within the context keep their speed, those below once are slowed down; the borders
    # lie at whole pairs, outwards
    def pair(b):
        return n_rot * math.log(ctx / (b * 2 * math.pi)) / (2 * math.log(base))
    low, high = max(0, math.floor(pair(32))), min(n_rot - 1, math.ceil(pair(1)))
    fast, slow = i <= low, i >= high
    assert np.allclose(got[fast], plain[fast], rtol=1e-14) and np.allclose(got[slow], plain[slow] / factor, rtol=1e-14)
    mix = np.clip((i - low) / max(0.001, high - low), 0, 1)
    assert np.allclose(got, plain / factor * mix + plain * (1 - mix), rtol=1e-14)
    assert (np.diff(got) < 0).all() and ((got >= plain / factor * (1 - 1e-14)) & (got <= plain * (1 + 1e-14))).all()
    assert (turns[fast][:-1] >= 32).all() if fast.sum() > 1 else True
    assert abs(scale - (1 + 0.1 * math.log(factor))) < 1e-6
    other, _ = kc.rope_freqs(n_rot, base, factor, yarn_ctx=ctx, beta_fast=32.0, beta_slow=1.0)
    assert np.array_equal(got, other)


def test_freqs_refused():
    for kw in (dict(n_rot=0), dict(n_rot=3), dict(n_rot=-2), dict(n_rot=1026), dict(base=1.0), dict(base=float("nan")), dict(base=float("inf")), dict(factor=0.0),
               dict(factor=-1.0), dict(factor=float("inf")), dict(yarn_ctx=-1), dict(beta_fast=-1.0), dict(beta_slow=float("nan"))):
        with pytest.raises(kc.KcError, match="InvalidValue"):
            kc.rope_freqs(**{**dict(n_rot=64, base=1e4), **kw})
    s = kc.RopeScaling(64, 1e4, 1.0, 0, 0.0, 0.0)
    out, f = np.zeros(32), C.c_float()
    L = kc.lib()
    assert L.kcRopeFreqs(None, None, out.ctypes.data, C.byref(f)) == L.kcRopeFreqs(C.byref(s), None, None, C.byref(f)) == kc.ERR["InvalidValue"]
    assert L.kcRopeFreqs(C.byref(s), None, out.ctypes.data, None) == kc.ERR["InvalidValue"]
    with pytest.raises(ValueError):
        kc.rope_freqs(64, 1e4, ff=np.ones(31))


# ---- the plain forms themselves, by hand

def test_plain_forms():
    got = plain_pages([5, 16, 0], [12, 1, 0], [9, 8, 7], np.array([[3, -1], [4, -1], [-1, -1]], np.int32), 16, 20, [-1] + [0] * 11 + [-1] + [0] * 7, 1)
    assert got["start"].tolist() == [0, 12, 13, 13] and got["len"].tolist() == [17, 17, 0] and got["used"] == 2
    assert got["table"].tolist() == [[3, 9], [4, 8], [-1, -1]]
    assert got["slots"].tolist() == [53, 54, 55, 56, 57, 58, 59, 60, 61, 62, 63, 144, 128] + [-1] * 7
    assert got["pos"].tolist() == [5] + [6] * 11 + [16] + [0] * 7 and got["tree"][:4, 0].tolist() == [1, 3, 5, 9]
    l = np.array([np.log(0.1), np.log(0.5), -np.inf, np.log(0.15), np.log(0.25)], np.float32)
    assert [plain_sample(l, u)[0][0] for u in (0.0, 0.49, 0.51, 0.74, 0.76, 0.89, 0.91, 1.0)] == [1, 1, 4, 4, 3, 3, 0, 0]
    assert plain_sample(l, 0.999, top_k=2)[0] == [4] and plain_sample(l, 0.999, top_p=0.5001)[0] == [4] and plain_sample(l, 0.999, top_p=0.49)[0] == [1]
    assert plain_sample(l, 0.999, min_p=0.4)[0] == [4] and plain_sample(l, 0.999, min_p=0.25)[0] == [3] and plain_sample(l, 0.999, temperature=0.0)[0] == [1]
    assert abs(plain_sample(l, 0.999, min_p=0.4)[1][0] - 1 / 3) < 1e-6
