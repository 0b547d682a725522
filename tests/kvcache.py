"""Plain forms, in 64 bits, of the operators over a key/value cache, and the calls the tests make of the kernels."""
import math

import numpy as np

import kernelcore_amd as kc


# ---- 4-bit blocks -------------------------------------------------------------------------------------------------

def pack_q4(x):
    """Rows of f32 values (..., n) as Q4_0 blocks (..., n / 32 * 18) bytes, codes decided in exact arithmetic: x / d in 64
    bits may round across a border, so a border is compared as a product (29 bits) instead."""
    x = np.asarray(x, np.float32).reshape(*np.shape(x)[:-1], np.shape(x)[-1] // 32, 32)
    at = np.abs(x).argmax(-1)[..., None]  # (numpy: the first of several)
    d = np.take_along_axis(x, at, -1) / np.float32(-8)
    a, y = np.abs(d).astype(np.float64), x.astype(np.float64) * np.sign(d)
    c = sum(((k - 8.5) * a <= y).astype(np.uint8) for k in range(1, 16))
    c = np.where(a == 0, np.uint8(8), c).astype(np.uint8)
    wild = ~np.isfinite(x).all(-1)
    c[wild] = 8
    with np.errstate(over="ignore"):
        h = d.astype(np.float16)
    h[wild] = np.nan
    return np.concatenate([h.view(np.uint8), c[..., :16] | (c[..., 16:] << 4)], -1).reshape(*x.shape[:-2], x.shape[-2] * 18)


def unpack_q4(b):
    """The values of blocks, in 64 bits."""
    b = np.asarray(b, np.uint8)
    b = b.reshape(*b.shape[:-1], b.shape[-1] // 18, 18)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    c = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float64) - 8
    with np.errstate(invalid="ignore"):
        return (d * c).reshape(*b.shape[:-2], b.shape[-2] * 32)


# ---- attention ----------------------------------------------------------------------------------------------------

class Case:
    """One call: q [N][H][D] f32; k, v as stored ([T][H_kv][...] fp16 or blocks); shaping; everything drawn from the seed."""

    def __init__(self, q4, H, H_kv, D, N, T, causal=1, prefix=0, cap=0.0, bias=False, docs=0, mask=None, kpos=None, qpos=None,
                 pos0=None, scale=None, seed=0, spread=1.0):
        r = np.random.default_rng([seed, D, N, T, H])
        self.q4, self.H, self.K, self.D, self.N, self.T = q4, H, H_kv, D, N, T
        self.causal, self.prefix, self.cap = causal, prefix, cap
        self.scale = 1.0 / math.sqrt(D) if scale is None else scale
        self.q = (r.standard_normal((N, H, D)) * spread).astype(np.float32)
        k, v = r.standard_normal((T, H_kv, D)).astype(np.float32), r.standard_normal((T, H_kv, D)).astype(np.float32)
        self.k, self.v = (pack_q4(k), pack_q4(v)) if q4 else (k.astype(np.float16), v.astype(np.float16))
        self.slopes = (2.0 ** (-8.0 * np.arange(1, H + 1) / H)).astype(np.float32) if bias else None
        self.pos0 = max(0, T - N) if pos0 is None else pos0
        self.qpos, self.kpos, self.mask = qpos, kpos, mask
        self.kdoc = self.qdoc = None
        if docs:
            self.kdoc = np.sort(r.integers(0, docs, T)).astype(np.int32)
            self.qdoc = self.kdoc[T - N:].copy() if N <= T else r.integers(0, docs, N).astype(np.int32)

    def values(self, x):
        return unpack_q4(x) if self.q4 else x.astype(np.float64)

    def scores(self):
        """(scores, seen, terms): [N][H][T]; terms: what a score's sum is made of, in magnitude."""
        N, H, K, T = self.N, self.H, self.K, self.T
        k = np.repeat(self.values(self.k), H // K, axis=1)
        q = self.q.astype(np.float64)
        with np.errstate(invalid="ignore", over="ignore"):
            x = np.stack([q[:, h] @ k[:, h].T for h in range(H)], 1) * np.float64(np.float32(self.scale))
            terms = np.stack([np.abs(q[:, h]) @ np.abs(k[:, h]).T for h in range(H)], 1) * abs(self.scale)
            if self.cap:
                x = self.cap * np.tanh(x / self.cap)
        i = (self.qpos if self.qpos is not None else self.pos0 + np.arange(N))[:, None, None]
        j = self.kpos if self.kpos is not None else np.arange(T)[None]
        j = np.broadcast_to(np.repeat(np.broadcast_to(j, (K, T)), H // K, axis=0)[None], (N, H, T))
        if self.slopes is not None:
            b = self.slopes[None, :, None].astype(np.float64) * np.abs(i - j)
            x, terms = x - b, terms + b
        seen = j >= 0
        if self.mask is not None:
            m = self.mask[:, None, :T].astype(np.float64)
            with np.errstate(invalid="ignore"):
                x = x + m
            seen = seen & ~(m == -np.inf)
            terms = terms + np.where(np.isfinite(m), np.abs(m), 0.0)
        if self.causal:
            seen = seen & ((j <= i) | (j < self.prefix))
        if self.kdoc is not None:
            kd = np.repeat(np.broadcast_to(self.kdoc, (K, T)), H // K, axis=0)
            seen = seen & (self.qdoc[:, None, None] == kd[None])
        return np.where(seen, x, -np.inf), seen, np.where(seen, terms, 0.0)

    def score_error(self, terms):
        """What the f32 arithmetic of a score may be off: products of split q within 2^-21 of the terms, a random walk of D
        f32 additions, ten roundings of the shaping that follows (tanh's relative error of 3e-7 < 5 2^-24 among them)."""
        top = float(terms.max()) if terms.size else 0.0
        return top * (2.0 ** -21 + (math.sqrt(self.D) + 10) * 2.0 ** -24)

    def expected(self):
        """(out, bound on |difference|, lse, its bound)"""
        N, H, K, T, D = self.N, self.H, self.K, self.T, self.D
        x, seen, terms = self.scores()
        v = np.repeat(self.values(self.v), H // K, axis=1)
        any_ = seen.any(-1)
        top = np.where(any_, np.max(np.where(seen, x, -np.inf), -1, initial=-np.inf), 0.0)
        p = np.where(seen, np.exp(x - top[..., None]), 0.0)
        total = p.sum(-1)
        w = p / np.where(any_, total, 1.0)[..., None]
        safe = np.where(np.isfinite(v), v, 0.0)
        out = np.stack([w[:, h] @ safe[:, h] for h in range(H)], 1)
        mag = np.stack([w[:, h] @ np.abs(safe[:, h]) for h in range(H)], 1)
        err = self.score_error(terms)
        bound = (2 * err + 2.0 ** -20 + 4 * math.sqrt(max(T, 1)) * 2.0 ** -24) * mag
        # each p (the largest between 1 and 16, so the sum at least 1) is two fp16 parts of 2^11 p, of which the second is a
        # multiple of 2^-24: off by up to half of that where it is subnormal, 2^-25 2^-11 = 2^-36
        bound += 2.0 ** -36 * np.stack([seen[:, h].astype(np.float64) @ np.abs(safe[:, h]) for h in range(H)], 1)
        lse = np.where(any_, top + np.log(np.where(any_, total, 1.0)), -np.inf)
        lse_bound = err + 2.0 ** -20 + 4 * math.sqrt(max(T, 1)) * 2.0 ** -24 + 2.0 ** -22 * np.abs(np.where(any_, lse, 0.0))
        return out, bound, lse, lse_bound

    def expected_weights(self, lse, w_in, decay):
        """(weights, bound) of [H_kv][T] for the given f32 lse"""
        x, seen, terms = self.scores()
        z = lse.astype(np.float64)[..., None]
        p = np.where(seen & (z > -np.inf), np.exp(np.where(seen & (z > -np.inf), x - z, 0.0)), 0.0)
        s = p.reshape(self.N, self.K, -1, self.T).sum((0, 2))
        zmax = float(np.abs(lse[np.isfinite(lse)]).max(initial=0.0))
        err = self.score_error(terms) + 2.0 ** -22 * zmax + 2.0 ** -20 + 4 * math.sqrt(self.N * self.H) * 2.0 ** -24
        base = 0.0 if w_in is None else np.float64(np.float32(decay)) * w_in.astype(np.float64)
        # (a weight below f32's smallest normal value, 2^-126, may come out as 0)
        return base + s, err * s + 2.0 ** -23 * np.abs(base + s) + self.N * self.H * 2.0 ** -126

    # ---- the calls

    def upload(self):
        """Device buffers by name (those that the case has)."""
        out = {}
        for name in ("q", "k", "v", "mask", "qpos", "kpos", "qdoc", "kdoc", "slopes"):
            a = getattr(self, name)
            if a is not None:
                a = np.ascontiguousarray(a, np.int32 if name in ("qpos", "kpos", "qdoc", "kdoc") else None)
                out[name] = kc.Buffer.of(a) if a.nbytes else kc.Buffer(16)
        return out

    def head_bytes(self):
        return self.D // 32 * 18 if self.q4 else 2 * self.D

    def dims(self, **over):
        hb = self.head_bytes()
        d = dict(H=self.H, H_kv=self.K, D=self.D, N=self.N, T=self.T, q_tok=self.H * self.D, q_head=self.D,
                 m_row=self.mask.shape[1] // 2 if self.mask is not None else 0,
                 key_row=self.T if self.kpos is not None and self.kpos.ndim == 2 and self.kpos.shape[0] > 1 else 0,
                 pos0=self.pos0, causal=self.causal, prefix=self.prefix, k_row=self.K * hb, k_head=hb, v_row=self.K * hb, v_head=hb)
        d.update(over)
        return kc.FlashExtDims(**d)

    def name(self, op):
        return op + ("_q4_0" if self.q4 else "_f16")

    def shape_args(self, b, d):
        p = {n: b[n].ptr for n in ("q", "k", "mask", "qpos", "kpos", "qdoc", "kdoc", "slopes") if n in b}
        return dict(p, d=d, scale=self.scale, softcap=self.cap)

    def attend(self, stream=None, lse=True):
        """(out, lse) of flash_ext; guard words after out and part must stay as they were."""
        b, d = self.upload(), self.dims()
        n, h = self.N * self.H * self.D, self.N * self.H
        part_bytes = kc.flash_ext_part_bytes(d)
        guard = np.full(64, 0x5A5A5A5A, np.uint32)
        out, sums, part = kc.Buffer(4 * n + 256), kc.Buffer(4 * h + 256), kc.Buffer(part_bytes + 256)
        for buf, at in ((out, 4 * n), (sums, 4 * h), (part, part_bytes)):
            buf.upload(guard, at)
        kc.launch(self.name("flash_ext"), kc.FlashExtArgs(v=b["v"].ptr, out=out.ptr, lse=sums.ptr if lse else None,
                                                          part=part.ptr if part_bytes else None, **self.shape_args(b, d)), stream)
        kc.synchronize()
        got = out.download(np.float32, n).reshape(self.N, self.H, self.D), sums.download(np.float32, h).reshape(self.N, self.H)
        for buf, at in ((out, 4 * n), (sums, 4 * h), (part, part_bytes)):
            assert (buf.download(np.uint32, 64, at) == guard).all()
        for x in [out, sums, part, *b.values()]:
            x.free()
        return got

    def weights(self, lse, w_in=None, decay=0.0):
        b, d = self.upload(), self.dims()
        bl, w = kc.Buffer.of(lse.astype(np.float32)), kc.Buffer(4 * self.K * self.T + 256)
        guard = np.full(64, 0x5A5A5A5A, np.uint32)
        w.upload(guard, 4 * self.K * self.T)
        bw = kc.Buffer.of(w_in.astype(np.float32)) if w_in is not None else None
        kc.launch(self.name("attn_weights"), kc.AttnWeightsArgs(lse=bl.ptr, w_in=bw.ptr if bw else None, w=w.ptr, w_row=self.T,
                                                                decay=decay, **self.shape_args(b, d)))
        kc.synchronize()
        got = w.download(np.float32, self.K * self.T).reshape(self.K, self.T)
        assert (w.download(np.uint32, 64, 4 * self.K * self.T) == guard).all()
        for x in [bl, w, *b.values()] + ([bw] if bw else []):
            x.free()
        return got

    def check(self):
        out, sums = self.attend()
        want, bound, lse, lse_bound = self.expected()
        bad = ~(np.abs(out - want) <= bound)
        assert not bad.any(), (np.argwhere(bad)[:4].tolist(), float(np.abs(out - want)[bad].max()), float(bound[bad].min()))
        assert (np.isneginf(sums) == np.isneginf(lse)).all()
        fin = np.isfinite(lse)
        assert (np.abs(sums[fin] - lse[fin]) <= lse_bound[fin]).all()
        assert (out[~fin] == 0).all()
        return out, sums
