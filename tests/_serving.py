"""Shared by the tests of the serving operators: device arrays, page layouts, and the operators'
definitions in float64."""
from __future__ import annotations

import numpy as np

from moe_mi355x.moe import read_device

DT = {"float32": np.float32, "float16": np.float16, "int8": np.int8}


class Arrays:
    """Device copies of NumPy arrays, freed together."""

    def __init__(self, backend, stream):
        self.backend, self.stream, self.held = backend, stream, []

    def put(self, a):
        a = np.ascontiguousarray(a)
        buf = self.backend.alloc_device(max(a.nbytes, 16))
        self.held.append(buf)
        if a.nbytes:
            self.backend.copy_h2d_ptr_async(buf.handle, a.ctypes.data, a.nbytes, self.stream)
            self.backend.synchronize_stream(self.stream)
        return int(buf.handle)

    def get(self, ptr, like):
        return read_device(self.backend, ptr, like.dtype, like.size, self.stream).reshape(like.shape)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.backend.synchronize_stream(self.stream)
        for b in self.held:
            self.backend.free_device(b)


class Batch:
    """A ragged batch over randomly placed pages.  ``news`` and ``lens``: new rows and cached
    tokens of every sequence; ``pad`` rows follow the last sequence's."""

    def __init__(self, rng, news, lens, page, spare=3, pad=0, extra_pages=0):
        self.news, self.lens, self.page = list(news), list(lens), page
        per = [-(-c // page) for c in lens]
        self.max_pages = max([1, *per]) + extra_pages
        self.n_pages = sum(per) + spare
        ids = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(per), self.max_pages), -1, dtype=np.int32)
        at = 0
        for b, p in enumerate(per):
            self.table[b, :p] = ids[at:at + p]
            at += p
        self.q_start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.kv_len = np.array(lens, dtype=np.int32)
        self.used = int(self.q_start[-1])
        self.rows = self.used + pad
        self.max_q, self.max_kv = max([1, *news]), max([0, *lens])

    def device(self, arrays):
        from moe_mi355x.paged_kv import paged_batch

        return paged_batch(arrays.put(self.q_start), arrays.put(self.kv_len),
                           arrays.put(self.table), n_seqs=len(self.news),
                           max_pages=self.max_pages, rows=self.rows, max_q=self.max_q,
                           max_kv=self.max_kv)

    def positions(self, b):
        return np.arange(self.lens[b] - self.news[b], self.lens[b])

    def slots(self, b, n_pages):
        """(page, row) of every cached token of sequence b, and which of them have a page."""
        j = np.arange(self.lens[b])
        pi = j // self.page
        page = np.where(pi < self.max_pages, self.table[b, np.minimum(pi, self.max_pages - 1)], -1)
        return page, j % self.page, (page >= 0) & (page < n_pages)


def pool_of(rng, batch, n_kv, hd, dtype, std=1.0, hole=np.nan):
    """A pool [pages, kv heads, page, hd] (and int8 scales) whose rows that no sequence holds are
    ``hole`` (int8: scales of NaN)."""
    shape = (batch.n_pages, n_kv, batch.page, hd)
    live = np.zeros((batch.n_pages, batch.page), bool)
    for b in range(len(batch.news)):
        page, row, ok = batch.slots(b, batch.n_pages)
        live[page[ok], row[ok]] = True
    x = rng.standard_normal(shape).astype(np.float32) * np.float32(std)
    mask = live[:, None, :, None]
    if dtype == "int8":
        scale = (np.abs(x).max(-1) / 127).astype(np.float32)
        q = np.clip(np.rint(x / scale[..., None]), -127, 127).astype(np.int8)
        return q, np.where(live[:, None], scale, np.float32(hole)).astype(np.float32)
    return np.where(mask, x, np.float32(hole)).astype(DT[dtype]), None


def values(pool, scale):
    return pool.astype(np.float64) * (1.0 if scale is None else scale[..., None].astype(np.float64))


def attention(batch, q, k, v, n_kv, scale, gate=None):
    """(outputs, sum of p |v|, largest |v|) per row in float64; k, v are pools of values."""
    rows, nh, hd = q.shape
    out, mag = np.zeros((rows, nh, hd)), np.zeros((rows, nh, hd))
    big = np.zeros((rows, nh, 1))
    n_pages = k.shape[0]
    for b, m in enumerate(batch.news):
        page, row, ok = batch.slots(b, n_pages)
        pos = batch.positions(b)
        r = slice(batch.q_start[b], batch.q_start[b] + m)
        if not m or not ok.any():
            continue
        j = np.nonzero(ok)[0]
        for h in range(nh):
            kv = h // (nh // n_kv)
            kk, vv = k[page[ok], kv, row[ok]], v[page[ok], kv, row[ok]]
            s = q[r, h].astype(np.float64) @ kk.T * scale
            s = np.where(j[None] <= pos[:, None], s, -np.inf)
            top = s.max(1, keepdims=True)
            p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
            tot = p.sum(1, keepdims=True)
            p = np.divide(p, tot, out=np.zeros_like(p), where=tot > 0)
            if np.isfinite(vv).all():
                out[r, h], mag[r, h], big[r, h] = p @ vv, p @ np.abs(vv), np.abs(vv).max()
                continue
            for i, t in enumerate(range(r.start, r.stop)):  # only what the row sees is multiplied
                see = j <= pos[i]
                out[t, h], mag[t, h] = p[i, see] @ vv[see], p[i, see] @ np.abs(vv[see])
                big[t, h] = np.abs(vv[see]).max() if see.any() else 0.0
    if gate is not None:
        g = 1.0 / (1.0 + np.exp(-gate.astype(np.float64)))
        out, mag = out * g, mag * g
    return out, mag, big


def rotated(x, w, pos, rotary, theta, eps):
    """Norm and rotary embedding of rows x [m, heads, hd] at positions pos, in float64."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    half = rotary // 2
    if not half:
        return x
    a = pos[:, None] * theta ** (-np.arange(half) / half)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    u, y = x[..., :half], x[..., half:rotary]
    return np.concatenate([u * c - y * s, y * c + u * s, x[..., rotary:]], -1)


def delta_rule(q, k, v, g, beta, state, scale, norm):
    """(o, state) of one sequence and one head, token by token in float64."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    if norm:
        q = q / np.sqrt((q * q).sum(-1, keepdims=True) + 1e-6)
        k = k / np.sqrt((k * k).sum(-1, keepdims=True) + 1e-6)
    s = np.array(state, dtype=np.float64)
    o = np.empty((len(q), s.shape[1]))
    for t in range(len(q)):
        s = s * np.exp(float(g[t]))
        s = s + np.outer(k[t], float(beta[t]) * (v[t] - k[t] @ s))
        o[t] = scale * (q[t] @ s)
    return o, s
