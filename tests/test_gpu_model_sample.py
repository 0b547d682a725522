"""kcModelSample against a loop of single-token forwards whose logits are drawn from by the definition in extended precision: the captured
step (decode, sample_rows, the step's bookkeeping) gives the same tokens and positions as the eager one, under changing cuts on one
model. Logits of both are the same bits (the same kernels on the same inputs), so tokens are compared exactly."""
import ctypes as C

import numpy as np
import pytest

import kernelcore_amd as kc
from tests import serve
from tests.model_weights import random_weights

pytestmark = pytest.mark.gpu

LLAMA = dict(n_layer=2, n_embd=512, n_head=8, n_head_kv=2, head_dim=64, n_ff=1024, n_vocab=1024, norm_eps=1e-5,
             rope_theta=500000.0, rope_neox=0, qk_norm=0, max_ctx=96, max_batch=64)
QWEN = dict(n_layer=1, n_embd=512, n_head=4, n_head_kv=2, head_dim=128, n_ff=768, n_vocab=1536, norm_eps=1e-6,
            rope_theta=1000000.0, rope_neox=1, qk_norm=1, max_ctx=96, max_batch=64)


@pytest.fixture(scope="module", autouse=True)
def runtime():
    kc.init()
    yield
    kc.synchronize()


def build(cfg, seed):
    m = kc.Model(**cfg)
    for (tid, layer), data in random_weights(cfg, seed).items():
        m.set_tensor(tid, layer, data)
    return m


@pytest.mark.parametrize("cfg", [LLAMA, QWEN], ids=["llama", "qwen3"])
def test_sample_matches_forward_loop(cfg):
    a, b = build(cfg, 5), build(cfg, 5)
    rng = np.random.default_rng(6)
    prompt = rng.integers(0, cfg["n_vocab"], 20)
    a.forward(prompt, want_logits=False)
    logits = b.forward(prompt)
    at = prompt.size
    for cuts in (dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.05), dict(temperature=1.5), dict(top_p=0.5), dict(top_k=3),
                 dict(temperature=0.0, top_k=7)):
        us = rng.random(7).astype(np.float32)
        us[0] = 0.999
        got = a.sample(us, **cuts)
        for i, u in enumerate(us):
            want, _ = serve.plain_sample(logits, u, **cuts)
            assert got[i] in want, (cuts, i, got, want)
            logits = b.forward([int(got[i])]) if i + 1 < us.size else logits
        at += us.size - 1
        assert a.position() == at == b.position()
        # (a call starts from the logits of the last position: the last token drawn is not in the cache)
    a.close()
    b.close()


def test_temperature_zero_is_generate():
    a, b = build(LLAMA, 8), build(LLAMA, 8)
    for m in (a, b):
        m.forward(np.arange(30, 50), want_logits=False)
    want = b.generate(12)
    assert list(a.sample(np.full(12, 0.7), temperature=0.0)) == list(want)
    assert a.position() == b.position()
    a.close()
    b.close()


def test_sample_and_generate_take_turns():
    """Both graphs of one model, with a reset between: neither leaves anything that the other takes for its own."""
    m = build(LLAMA, 9)
    us = np.linspace(0.05, 0.95, 9, dtype=np.float32)
    first = None
    for _ in range(3):
        m.reset()
        m.forward(np.arange(5, 25), want_logits=False)
        s = list(m.sample(us, temperature=1.2, top_p=0.9))
        g = list(m.generate(6))
        s2 = list(m.sample(us[:1]))
        first = first or (s, g, s2)
        assert (s, g, s2) == first
    m.close()


def test_refusals():
    m = build(dict(LLAMA, n_layer=1), 3)
    how, us, out = kc.ModelSampling(1.0, 0, 1.0, 0.0), (C.c_float * 8)(), (C.c_int * 8)()
    L = kc.lib()

    def err(*args):
        return kc.ERRORS[L.kcModelSample(*args)]
    assert err(m.h, C.byref(how), us, 4, out) == "InvalidValue"  # nothing forwarded
    m.forward([1, 2, 3], want_logits=False)
    assert err(m.h, None, us, 4, out) == "InvalidValue"
    assert err(m.h, C.byref(how), None, 4, out) == "InvalidValue"
    assert err(m.h, C.byref(how), us, 0, out) == "InvalidValue"
    assert err(m.h, C.byref(how), us, LLAMA["max_ctx"], out) == "InvalidValue"
    assert err(m.h, C.byref(how), us, 4097, out) == "InvalidValue"
    assert m.position() == 3
    assert L.kcModelSample(m.h, C.byref(how), us, 1, None) == 0
    m.close()
