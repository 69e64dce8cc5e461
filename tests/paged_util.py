"""A plain model of the paged KV cache: pools as numpy bytes in the library's page
layout, rows decoded and encoded element by element, and the batch's attention
in float64."""
import math

import numpy as np

F32, F16, Q4_0, Q8_0 = 0, 1, 2, 8


def row_bytes(t, hd):
    return 2 * hd if t == F16 else hd if t == Q8_0 else hd // 2


def page_bytes(t, n_kv, hd, page):
    return n_kv * page * (row_bytes(t, hd) + (0 if t == F16 else hd // 16))


def quantize(t, x):
    """(quants, fp16 scales) of rows of float32 in blocks of 32, in the cache's fp32 arithmetic."""
    b = x.astype(np.float32).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    if t == Q8_0:
        top = np.abs(b).max(-1, keepdims=True)
        inv = np.divide(np.float32(127), top, out=np.zeros_like(top), where=top != 0)
        return np.rint(b * inv).astype(np.int32), (top * np.float32(1 / 127.0)).astype(np.float16)[..., 0]
    i = np.abs(b).argmax(-1)[..., None]
    d = np.take_along_axis(b, i, -1) * np.float32(-0.125)
    inv = np.divide(np.float32(1), d, out=np.zeros_like(d), where=d != 0)
    # x * inv + 8.5 with one rounding, truncated
    q = np.trunc((b.astype(np.float64) * inv + 8.5).astype(np.float32)).astype(np.int32)
    return np.minimum(q, 15) - 8, d.astype(np.float16)[..., 0]


def values(t, x):
    """The values a cache of type t holds for rows x (float64)."""
    if t == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float32).astype(np.float16).astype(np.float64)
    q, d = quantize(t, x)
    return (q * d.astype(np.float64)[..., None]).reshape(x.shape)


class Pool:
    """Keys and values of `n_pages` pages as the library lays them out."""

    def __init__(self, t, n_kv, hd, page, n_pages, fill=0):
        self.t, self.n_kv, self.hd, self.page, self.n_pages = t, n_kv, hd, page, n_pages
        self.pb = page_bytes(t, n_kv, hd, page)
        self.k = np.full((n_pages, self.pb), fill, np.uint8)
        self.v = np.full((n_pages, self.pb), fill, np.uint8)
        e = np.arange(hd)
        s, g, j, m, c = e // 32, e % 32 // 8, e % 8, e // 16, e % 16
        self.k8, self.v8 = g * (hd // 4) + 8 * s + j, c * (hd // 16) + m
        self.k4 = 8 * (g * (hd // 32) + s) + (j >> 1) + 4 * (j & 1)
        self.v4 = c * (hd // 16) + m

    def put(self, value, pg, slot, h, x):
        """One row (float32 [hd])."""
        raw, row, hd = (self.v if value else self.k)[pg], h * self.page + slot, self.hd
        n = row_bytes(self.t, hd)
        if self.t == F16:
            with np.errstate(over="ignore"):
                raw[row * n:(row + 1) * n] = x.astype(np.float16).view(np.uint8)
            return
        q, d = quantize(self.t, x)
        q = q.reshape(-1)
        out = np.zeros(n, np.uint8)
        if self.t == Q8_0:
            out[self.v8 if value else self.k8] = q + 128
        else:
            nib = np.zeros(hd, np.uint8)
            nib[self.v4 if value else self.k4] = q + 8
            out = nib[0::2] | (nib[1::2] << 4)
        raw[row * n:(row + 1) * n] = out
        at = self.n_kv * self.page * n + row * (hd // 16)
        raw[at:at + hd // 16] = d.view(np.uint8)

    def get(self, value, pg, slot, h):
        raw, row, hd = (self.v if value else self.k)[pg], h * self.page + slot, self.hd
        n = row_bytes(self.t, hd)
        b = raw[row * n:(row + 1) * n]
        if self.t == F16:
            return b.view(np.float16).astype(np.float64)
        at = self.n_kv * self.page * n + row * (hd // 16)
        d = raw[at:at + hd // 16].view(np.float16).astype(np.float64)
        if self.t == Q8_0:
            q = b[self.v8 if value else self.k8].astype(np.float64) - 128
        else:
            nib = np.stack([b & 15, b >> 4], -1).reshape(-1)
            q = nib[self.v4 if value else self.k4].astype(np.float64) - 8
        return q * np.repeat(d, 32)


def turn(x, pos, n_rot, base, interleaved=False, factors=None):
    """RoPE of rows x [tokens][heads][hd] at positions pos, in float64."""
    y = x.astype(np.float64).copy()
    half = n_rot // 2
    i = np.arange(half)
    ang = np.asarray(pos, np.float64)[:, None] * base ** (-2.0 * i / max(n_rot, 1))
    if factors is not None:
        ang = ang / factors.astype(np.float64)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def attend(q, keys, vals, pos, scale, cap=0.0, window=0):
    """One (token, head): q [hd] at position pos over keys / vals [n][hd]; the
    output and its tolerance, both float64.

    The tolerance counts the roundings of an fp32 computation: a query and a
    weight enter as two truncated halves (2^-21 each), sums of hd products in
    fp32 (hd 2^-24 of the sum of magnitudes), the scaled score and its
    exponential (2^-22 of the score and 2^-22), tanh (cap 2^-21), the weighted
    sum over n positions (n 2^-24 at worst, here 2^-18, far above what n random
    roundings give) -- a score off by d moves a weight by d (1 + d), numerator
    and denominator both.  A weight's low half has steps of 2^-24, of 2^6 for the
    row's largest weight (quantized: of weight times scale, against the largest
    such product and its scale's power of two, so at most 2 more): what lies
    below 2^-30 of the largest is cut, 2^-29 of it from each of n positions, times
    a value of at most the largest."""
    lo = max(0, pos + 1 - window) if window else 0
    if pos < 0:
        return np.zeros_like(q, dtype=np.float64), np.zeros(len(q))
    k, v = keys[lo:pos + 1], vals[lo:pos + 1]
    with np.errstate(invalid="ignore", over="ignore"):
        s = k @ q.astype(np.float64) * scale
        size = np.abs(k) @ np.abs(q.astype(np.float64)) * abs(scale)
        if cap:
            s = cap * np.tanh(s / cap)
        d = size.max() * (2.0 ** -21 + len(q) * 2.0 ** -24) + np.abs(s).max() * 2.0 ** -22 + cap * 2.0 ** -21 + 2.0 ** -22
        w = np.exp(s - s.max())
        out = (w[:, None] * v).sum(0) / w.sum()
        mag = (w[:, None] * np.abs(v)).sum(0) / w.sum()
        cut = 2.0 ** -29 * len(v) * np.abs(v).max() * w.max() / w.sum()
    return out, (2 * d + 2.0 ** -18) * mag + cut + 1e-30


class Case:
    """A batch over a paged cache on the device, its plain twin beside it."""

    def __init__(self, G, t, n_head, n_kv, hd, page, lens, new=None, pad=0, n_prefix=0, seed=0, spread=1.0, poison=True):
        self.G, self.t, self.n_head, self.n_kv, self.hd, self.page = G, t, n_head, n_kv, hd, page
        self.lens, self.new = list(lens), list(new) if new is not None else [1] * len(lens)
        self.n_prefix, self.pad = n_prefix, pad
        rng = self.rng = np.random.default_rng(seed)
        self.n_tok = sum(self.new) + pad
        self.max_len = max(self.lens, default=0)
        need = [-(-n // page) for n in self.lens]
        n_pre = -(-n_prefix // page)
        n_pages = sum(need) + n_pre + 2
        ids = rng.permutation(n_pages).astype(np.int32)
        self.stride = max(need + [1])
        self.table = np.full((len(self.lens), self.stride), -7, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = ids[at:at + n]
            at += n
        self.prefix = ids[at:at + n_pre].copy()
        # what no position uses holds NaN scales / halves (0xff bytes)
        self.pool = Pool(t, n_kv, hd, page, n_pages, 0xff if poison else 0)
        self.rows = [self._fill(self.table[i], n, spread) for i, n in enumerate(self.lens)]
        self.shared = self._fill(self.prefix, n_prefix, spread)
        self.q = (rng.standard_normal((self.n_tok, n_head, hd)) * spread).astype(np.float32)
        self.one = new is None and not pad
        self.off = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self._upload()

    def _fill(self, pages, n, spread):
        k = (self.rng.standard_normal((n, self.n_kv, self.hd)) * spread).astype(np.float32)
        v = (self.rng.standard_normal((n, self.n_kv, self.hd)) * spread).astype(np.float32)
        for p in range(n):
            for h in range(self.n_kv):
                self.pool.put(False, pages[p // self.page], p % self.page, h, k[p, h])
                self.pool.put(True, pages[p // self.page], p % self.page, h, v[p, h])
        return [values(self.t, k), values(self.t, v)]

    def _upload(self):
        G, B = self.G, self.G.Buffer.from_array
        self.kv = G.PagedKV(self.t, self.n_kv, self.hd, self.page, self.pool.n_pages, k=B(self.pool.k), v=B(self.pool.v))
        self.d = dict(lens=B(np.asarray(self.lens + [0], np.int32)), table=B(self.table if self.table.size else np.zeros(1, np.int32)), off=B(self.off),
                      q=B(self.q if self.q.size else np.zeros(1, np.float32)))
        self.d["pre"] = B(self.prefix) if self.n_prefix else None
        self.batch = G.PagedBatch(len(self.lens), self.n_tok, self.d["lens"], self.d["table"], self.stride, self.max_len,
                                  q_off=None if self.one else self.d["off"], n_prefix=self.n_prefix, prefix=self.d["pre"])

    def attn(self, scale, cap=0.0, window=0, out=None, **more):
        G = self.G
        out = out or G.Buffer.from_array(np.full((max(1, self.n_tok), self.n_head, self.hd), 7.5, np.float32))
        G.paged_attn(self.kv, self.batch, self.d["q"], self.n_head, out, scale=scale, softcap=cap, window=window, **more)
        return out.download(np.float32, (self.n_tok, self.n_head, self.hd))

    def expect(self, scale, cap=0.0, window=0):
        """Outputs and tolerances; rows behind the last sequence keep 7.5."""
        grp = self.n_head // self.n_kv
        out, tol = np.full((self.n_tok, self.n_head, self.hd), 7.5), np.zeros((self.n_tok, self.n_head, self.hd))
        for s, (n, size) in enumerate(zip(self.new, self.lens)):
            for i in range(n):
                t, own = self.off[s] + i, size - n + i
                for h in range(self.n_head):
                    k, v = (np.concatenate([self.shared[w][:, h // grp], self.rows[s][w][:, h // grp]]) for w in (0, 1))
                    out[t, h], tol[t, h] = attend(self.q[t, h], k, v, self.n_prefix + own if own >= 0 else -1, scale, cap, window)
        return out, tol

    def check(self, scale=None, cap=0.0, window=0, **more):
        scale = self.hd ** -0.5 if scale is None else scale
        got = self.attn(scale, cap, window, **more).astype(np.float64)
        want, tol = self.expect(scale, cap, window)
        bad = ~(np.abs(got - want) <= tol) & ~(np.isnan(got) & np.isnan(want))
        worst = np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-30), initial=0.0)
        assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {worst:.3g} tolerances, first {tuple(np.argwhere(bad)[0])}"
        assert self.kv.status() == 0
        return worst


class LongCase(Case):
    """A Case of many rows: the same batch, filled and attended array by array."""

    def _fill(self, pages, n, spread):
        out = []
        for value in (False, True):
            x = (self.rng.standard_normal((n, self.n_kv, self.hd), np.float32) * np.float32(spread)).astype(np.float32)
            raw, pos, hd = self.pool.v if value else self.pool.k, np.arange(n), self.hd
            size = row_bytes(self.t, hd)
            rows = raw[:, :self.n_kv * self.page * size].reshape(len(raw), self.n_kv, self.page, size)
            at = (pages[pos // self.page][:, None], np.arange(self.n_kv), (pos % self.page)[:, None])
            if self.t == F16:
                rows[at] = x.astype(np.float16).view(np.uint8)
            else:
                q, d = quantize(self.t, x)
                q = q.reshape(x.shape)
                if self.t == Q8_0:
                    b = np.zeros(x.shape, np.uint8)
                    b[..., self.pool.v8 if value else self.pool.k8] = q + 128
                else:
                    b = np.zeros(x.shape, np.uint8)
                    b[..., self.pool.v4 if value else self.pool.k4] = q + 8
                    b = b[..., 0::2] | (b[..., 1::2] << 4)
                rows[at] = b
                raw[:, self.n_kv * self.page * size:].reshape(len(raw), self.n_kv, self.page, hd // 16)[at] = d.view(np.uint8)
            out.append(values(self.t, x))
        return out

    def expect(self, scale, cap=0.0, window=0):
        """As Case.expect; a row's tolerance takes the largest value up to its position."""
        grp, hd = self.n_head // self.n_kv, self.hd
        out, tol = np.full((self.n_tok, self.n_head, hd), 7.5), np.zeros((self.n_tok, self.n_head, hd))
        for s, (n, size) in enumerate(zip(self.new, self.lens)):
            own = size - n + np.arange(n)
            pos = np.where(own >= 0, self.n_prefix + own, -1)
            for kv in range(self.n_kv if n else 0):
                k, v = (np.concatenate([self.shared[w][:, kv], self.rows[s][w][:, kv]]) for w in (0, 1))
                key = np.arange(len(k))
                seen = key <= pos[:, None]
                if window:
                    seen &= key > pos[:, None] - window
                top = np.concatenate([np.maximum.accumulate(np.abs(v).max(1)), [0.0]])[pos]
                for h in range(kv * grp, (kv + 1) * grp):
                    q = self.q[self.off[s]:self.off[s] + n, h].astype(np.float64)
                    x = q @ k.T * scale
                    mag = np.where(seen, np.abs(q) @ np.abs(k).T * abs(scale), 0.0).max(1, initial=0.0)
                    if cap:
                        x = cap * np.tanh(x / cap)
                    x = np.where(seen, x, -np.inf)
                    d = mag * (2.0 ** -21 + hd * 2.0 ** -24) + np.where(seen, np.abs(x), 0.0).max(1, initial=0.0) * 2.0 ** -22 + cap * 2.0 ** -21 + 2.0 ** -22
                    w = np.exp(x - x.max(1, initial=-1e300)[:, None])
                    total = np.maximum(w.sum(1), 1e-300)[:, None]
                    t = slice(self.off[s], self.off[s] + n)
                    out[t, h] = w @ v / total
                    tol[t, h] = (2 * d[:, None] + 2.0 ** -18) * (w @ np.abs(v)) / total + 2.0 ** -29 * (seen.sum(1) * top)[:, None] / total + 1e-30
        return out, tol
