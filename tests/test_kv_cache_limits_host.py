"""Limits of the cache operators' arguments, on the CPU: the library over a stand-in for the HIP runtime (tests/hip_stub)."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))

START = r"""
import ctypes as C, math, sys
stub = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
stub.stub_record.restype = C.c_char_p
import kernelcore_amd as kc
kc.init()


def status(name, args):
    stub.stub_clear()
    r = kc.launch_status(name, args)
    assert (stub.stub_record() != b"") == (r == "Success"), (name, r)  # refused before anything is launched
    return r


def buf(n):
    return kc.Buffer(n).ptr


"""

CAPS = r"""
for q4, t in ((False, "_f16"), (True, "_q4_0")):
    d = kc.FlashExtDims(H=2, H_kv=1, D=64, N=2, T=40, q_tok=128, q_head=64, pos0=38, causal=1, k_row=36 if q4 else 128, v_row=36 if q4 else 128)
    common = dict(q=buf(4 * 256), k=buf(40 * 128), lse=buf(16), d=d, scale=0.1)
    v, out, w = buf(40 * 128), buf(4 * 256), buf(160)
    part = buf(kc.flash_ext_part_bytes(d) + 4)
    for cap, want in ((0.0, "Success"), (2.0 ** -100, "Success"), (2.0 ** 100, "Success"), (30.0, "Success"), (2.0 ** -101, "InvalidValue"), (1e-44, "InvalidValue"),
                      (2.0 ** 101, "InvalidValue"), (3e38, "InvalidValue"), (-1.0, "InvalidValue"), (math.nan, "InvalidValue"), (math.inf, "InvalidValue")):
        assert status("flash_ext" + t, kc.FlashExtArgs(v=v, out=out, part=part, softcap=cap, **common)) == want, cap
        assert status("attn_weights" + t, kc.AttnWeightsArgs(w=w, w_row=40, softcap=cap, **common)) == want, cap
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    stub = str(tmp_path_factory.mktemp("stub") / "hip_stub.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", os.path.join(HERE, "hip_stub", "hip_stub.cpp"), "-o", stub],
                   check=True)

    def go(body):
        r = subprocess.run([sys.executable, "-c", START + body + 'print("done")\n', stub], capture_output=True, text=True, cwd=os.path.dirname(HERE), timeout=300)
        assert r.returncode == 0 and r.stdout.split() == ["done"], r.stdout + r.stderr

    return go


def test_caps(run):
    """Caps whose reciprocal or product with a score leaves f32 are refused."""
    run(CAPS)
