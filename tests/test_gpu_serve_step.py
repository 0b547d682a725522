"""Steps of several requests as a serving loop makes them: pages and slots from the requests' lengths, rotary positions with the store into
the paged cache, attention of prompts, drafted trees and single tokens, logits, and a token drawn for every row -- each step against the
same in 64 bits from the operators' definitions, and as one captured graph."""
import ctypes as C

import numpy as np
import pytest

import kernelcore_amd as kc
from tests.serve import plain_pages, plain_sample, plain_turn, up

pytestmark = pytest.mark.gpu

H, K, D, PAGE, MAX_PAGES, SEQS, N, VOCAB, WORDS = 8, 2, 128, 16, 12, 4, 96, 1024, 3


@pytest.fixture(scope="module", autouse=True)
def runtime():
    kc.init()
    yield
    kc.synchronize()


class Server:
    """The device state of a serving loop, and its step's launches."""

    def __init__(self):
        r = np.random.default_rng(0)
        self.n_pages = SEQS * MAX_PAGES
        self.freqs, self.scale = kc.rope_freqs(D, 1e4, factor=4.0, yarn_ctx=64)
        self.head = (r.standard_normal((VOCAB, H * D)) * 0.05).astype(np.float16)
        self.b = {n: kc.Buffer(size) for n, size in dict(
            have=4 * SEQS, add=4 * SEQS, free=4 * self.n_pages, parent=4 * N, table=4 * SEQS * MAX_PAGES, start=4 * SEQS + 4, len=4 * SEQS, slots=8 * N, pos=4 * N,
            used=4, tree=4 * N * WORDS, q=4 * N * H * D, k=4 * N * K * D, v=4 * N * K * D, qr=4 * N * H * D, kc=self.n_pages * PAGE * K * D * 2,
            vc=self.n_pages * PAGE * K * D * 2, out=4 * N * H * D, logits=4 * N * VOCAB, u=4 * N, temperature=4 * N, top_k=4 * N, top_p=4 * N, tokens=4 * N,
            probs=4 * N).items()}
        self.b["freqs"], self.b["head"] = up(self.freqs, np.float64), up(self.head, np.float16)
        self.b["table"].upload(np.full((SEQS, MAX_PAGES), -1, np.int32))
        p = {n: x.ptr for n, x in self.b.items()}
        dims = kc.FlashPagesDims(H=H, H_kv=K, D=D, N=N, seqs=SEQS, page=PAGE, max_pages=MAX_PAGES, n_pages=self.n_pages, tree_words=WORDS, q_tok=H * D, q_head=D,
                                 table_row=MAX_PAGES, k_row=2 * K * D, k_head=2 * D, v_row=2 * K * D, v_head=2 * D)
        self.b["fpart"], self.b["spart"] = kc.Buffer(kc.flash_pages_part_bytes(dims)), kc.Buffer(kc.sample_rows_part_bytes(N, VOCAB))
        self.launches = [
            ("kv_pages", kc.KvPagesArgs(**{n: p[n] for n in ("have", "add", "free", "parent", "table", "start", "len", "slots", "pos", "used", "tree")}, seqs=SEQS,
                                        n_tokens=N, n_free=self.n_pages, page=PAGE, max_pages=MAX_PAGES, table_row=MAX_PAGES, tree_words=WORDS)),
            ("rope_ext", kc.RopeExtArgs(q=p["q"], k=p["k"], v=p["v"], pos=p["pos"], freqs=p["freqs"], slots=p["slots"], q_out=p["qr"], k_cache=p["kc"], v_cache=p["vc"],
                                        n_tokens=N, H=H, H_kv=K, D=D, n_rot=D, q_tok=H * D, q_head=D, k_tok=K * D, k_head=D, v_tok=K * D, v_head=D, out_tok=H * D,
                                        out_head=D, cache_rows=self.n_pages * PAGE, kc_row=2 * K * D, kc_head=2 * D, vc_row=2 * K * D, vc_head=2 * D, scale=self.scale)),
            ("flash_pages_f16", kc.FlashPagesArgs(q=p["qr"], k=p["kc"], v=p["vc"], table=p["table"], start=p["start"], len=p["len"], tree=p["tree"], out=p["out"],
                                                  part=self.b["fpart"].ptr, d=dims, scale=D ** -0.5)),
            ("matmul_f16", kc.MatmulF16Args(p["head"], p["out"], p["logits"], None, VOCAB, H * D, N)),
            ("sample_rows", kc.SampleRowsArgs(logits=p["logits"], u=p["u"], temperature=p["temperature"], top_k=p["top_k"], top_p=p["top_p"], tokens=p["tokens"],
                                              probs=p["probs"], part=self.b["spart"].ptr, row=VOCAB, rows=N, n_vocab=VOCAB))]
        # what a plain program keeps: every committed position's key and value
        self.keys = [np.zeros((0, K, D)) for _ in range(SEQS)]
        self.values = [np.zeros((0, K, D)) for _ in range(SEQS)]
        self.have = np.zeros(SEQS, np.int64)
        self.table = np.full((SEQS, MAX_PAGES), -1, np.int32)
        self.free = list(r.permutation(self.n_pages))

    def inputs(self, r, add, kind):
        """A step's inputs, on the host and on the device."""
        parent = np.full(N, -1, np.int64)
        at = 0
        for n in add:
            i = np.arange(n)
            parent[at:at + n] = i - 1 if kind == "prompt" else np.where(i == 0, -1, (r.random(n) * i).astype(int))
            at += n
        x = dict(have=self.have.astype(np.int32), add=np.asarray(add, np.int32), free=np.resize(np.array(self.free, np.int32), self.n_pages), parent=parent.astype(np.int32),
                 q=r.standard_normal((N, H, D)).astype(np.float32), k=r.standard_normal((N, K, D)).astype(np.float32), v=r.standard_normal((N, K, D)).astype(np.float32),
                 u=r.random(N).astype(np.float32), temperature=r.uniform(0.3, 1.2, N).astype(np.float32), top_k=r.choice([0, 5, 100], N).astype(np.int32),
                 top_p=r.choice([1.0, 0.9], N).astype(np.float32))
        for n, a in x.items():
            self.b[n].upload(a)
        return x

    def check(self, x, add):
        """The step's results from the definitions; commits what each request keeps of its tokens."""
        got = {n: self.b[n].download(t) for n, t in dict(slots=np.int64, pos=np.int32, tokens=np.int32, probs=np.float32, out=np.float32, logits=np.float32,
                                                         used=np.int32, table=np.int32).items()}
        want = plain_pages(self.have, add, x["free"], self.table, PAGE, N, x["parent"], WORDS)
        for n in ("slots", "pos", "used", "table"):
            assert np.array_equal(got[n].reshape(want[n].shape), want[n]), n
        self.table = want["table"]
        q, qb = plain_turn(x["q"], want["pos"], self.freqs, self.scale, D, False)
        k, _ = plain_turn(x["k"], want["pos"], self.freqs, self.scale, D, False)
        k, v = k.astype(np.float16).astype(np.float64), x["v"].astype(np.float16).astype(np.float64)
        out, logits = got["out"].reshape(N, H, D), got["logits"].reshape(N, VOCAB)
        for s in range(SEQS):
            a, b = want["start"][s:s + 2]
            if a == b:
                continue
            bits = (want["tree"][a:b].view(np.uint32)[:, :, None] >> np.arange(32, dtype=np.uint32) & 1).reshape(b - a, 32 * WORDS)[:, :b - a].astype(bool)
            seen = np.concatenate([np.ones((b - a, self.have[s]), bool), bits], 1)
            keys, values = np.concatenate([self.keys[s], k[a:b]]), np.concatenate([self.values[s], v[a:b]])
            for h in range(H):
                z = np.where(seen, q[a:b, h] @ keys[:, h // (H // K)].T * D ** -0.5, -np.inf)
                p = np.exp(z - z.max(1, keepdims=True))
                # a stored key may be one fp16 step off where its turned value lies next to a border: 2^-10 of 128 terms that average
                # out, in scores of a few units (below 2^-8), and twice that in the weights
                y = p / p.sum(1, keepdims=True) @ values[:, h // (H // K)]
                assert np.abs(out[a:b, h] - y).max(initial=0.0) < 2.0 ** -6
        live = int(want["start"][-1])
        ref = out[:live].reshape(live, -1).astype(np.float64) @ self.head.astype(np.float64).T
        # (fp16 weights times activations in two fp16 parts, f32 sums of 1024 terms)
        assert np.abs(logits[:live] - ref).max(initial=0.0) <= 2.0 ** -16 * np.abs(out[:live]).reshape(live, -1).sum(1).max(initial=1.0)
        for t in range(live):
            right, _ = plain_sample(logits[t], x["u"][t], float(x["temperature"][t]), int(x["top_k"][t]), float(x["top_p"][t]))
            assert got["tokens"][t] in right, t
        self.free = self.free[int(got["used"][0]):]
        return want, k, v

    def commit(self, add, want, k, v, keep):
        """Of each request's tokens the first keep[s] stay; pages past them go back to the free list."""
        for s in range(SEQS):
            a = want["start"][s]
            self.keys[s] = np.concatenate([self.keys[s], k[a:a + keep[s]]])
            self.values[s] = np.concatenate([self.values[s], v[a:a + keep[s]]])
            self.have[s] += keep[s]
            for p in range(-(-int(self.have[s]) // PAGE), -(-int(want["len"][s]) // PAGE)):
                self.free.append(int(self.table[s, p]))


STEPS = [("prompt", [40, 17, 1, 0]), ("tree", [10, 7, 24, 1]), ("tree", [1, 1, 1, 30]), ("prompt", [1, 50, 16, 15]), ("tree", [20, 1, 33, 9])]


def test_steps():
    r = np.random.default_rng(1)
    sv = Server()
    for kind, add in STEPS:
        x = sv.inputs(r, add, kind)
        for name, args in sv.launches:
            kc.launch(name, args)
        kc.synchronize()
        want, k, v = sv.check(x, add)
        sv.commit(add, want, k, v, add if kind == "prompt" else [min(1, n) for n in add])
    for b in sv.b.values():
        b.free()


def test_captured_step():
    """The whole step as one graph, launched for every step whatever the requests bring."""
    r = np.random.default_rng(2)
    sv = Server()
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
        want, k, v = sv.check(x, add)
        sv.commit(add, want, k, v, add if kind == "prompt" else [min(1, n) for n in add])
    kc.call("kcGraphDestroy", g)
    kc.call("kcStreamDestroy", s)
    for b in sv.b.values():
        b.free()
