"""The step of test_gpu_serve_step.py as one captured graph and launched one by one over the same inputs: the same bits in every output and in the
caches. And its attention against the 64-bit form over the cache as it is stored, within the bounds derived in tests/serve.py."""
import ctypes as C

import numpy as np
import pytest

import kernelcore_amd as kc
from tests.serve import Pages
from tests.test_gpu_serve_step import D, H, K, MAX_PAGES, N, PAGE, SEQS, STEPS, WORDS, Server

pytestmark = pytest.mark.gpu

OUTPUTS = dict(start=np.int32, len=np.int32, slots=np.int64, pos=np.int32, used=np.int32, tree=np.int32, qr=np.float32, kc=np.uint16, vc=np.uint16, out=np.float32,
               logits=np.float32, tokens=np.int32, probs=np.float32)


@pytest.fixture(scope="module", autouse=True)
def runtime():
    kc.init()
    yield
    kc.synchronize()


def outputs(sv):
    """Bits of everything that a step writes; of rows behind the last token what an output leaves as it was is left out."""
    got = {n: sv.b[n].download(t) for n, t in OUTPUTS.items()}
    got["table"] = sv.b["table"].download(np.int32)
    live = int(got["start"][SEQS])
    got["out"] = got["out"].reshape(N, -1)[:live]
    for n in ("logits", "tokens", "probs"):
        got[n] = got[n].reshape(N, -1)[:live]
    return got


def attention_case(sv, got):
    """The step's attention as a case of tests/serve.py, on what the cache holds."""
    c = Pages.__new__(Pages)
    c.H, c.K, c.D, c.page, c.words, c.scale = H, K, D, PAGE, WORDS, D ** -0.5
    c.start, c.lens = got["start"], got["len"].astype(np.int64)
    c.nodes, c.N, c.n_pages, c.max_pages = np.diff(c.start), int(got["start"][SEQS]), sv.n_pages, MAX_PAGES
    c.table = got["table"].reshape(SEQS, MAX_PAGES)
    c.q = got["qr"].reshape(N, H, D)[:c.N]
    c.k, c.v = (got[n].view(np.float16).reshape(-1, K, D) for n in ("kc", "vc"))
    c.tree = got["tree"].view(np.uint32).reshape(N, WORDS)
    return c


def test_captured_is_eager():
    r = np.random.default_rng(5)
    sv = Server()
    for n in ("kc", "vc"):
        sv.b[n].upload(np.zeros(sv.n_pages * PAGE * K * D, np.float16))
    sv.b["out"].upload(np.zeros(N * H * D, np.float32))
    s, g = C.c_void_p(), C.c_void_p()
    kc.call("kcStreamCreate", C.byref(s))
    kc.call("kcStreamBeginCapture", s)
    for name, args in sv.launches:
        kc.launch(name, args, s)
    kc.call("kcStreamEndCapture", s, C.byref(g))
    for kind, add in STEPS:
        x = sv.inputs(r, add, kind)
        kc.call("kcGraphLaunch", g, s)
        kc.synchronize()
        captured = outputs(sv)
        # the rows that the step stored, and its outputs, are made anew
        slots = captured["slots"][captured["slots"] >= 0]
        for n in ("kc", "vc"):
            scribbled = captured[n].reshape(-1, K * D).copy()
            scribbled[slots] = 0x5555
            sv.b[n].upload(scribbled)
        for n in ("start", "len", "slots", "pos", "used", "tree", "qr", "logits", "tokens", "probs"):
            size = sv.b[n].download(np.uint8).size
            sv.b[n].upload(np.full(size, 0xAA, np.uint8))
        sv.b["out"].upload(np.zeros(N * H * D, np.float32))
        for name, args in sv.launches:
            kc.launch(name, args)
        kc.synchronize()
        eager = outputs(sv)
        for n, a in captured.items():
            assert np.array_equal(a.view(np.uint8), eager[n].view(np.uint8)), (kind, add, n)
        c = attention_case(sv, captured)
        want, bound, _, _ = c.expected()
        assert (np.abs(captured["out"].reshape(c.N, H, D) - want) <= bound).all(), (kind, add)
        made, k, v = sv.check(x, add)
        sv.commit(add, made, k, v, add if kind == "prompt" else [min(1, n) for n in add])
    kc.call("kcGraphDestroy", g)
    kc.call("kcStreamDestroy", s)
    for b in sv.b.values():
        b.free()
