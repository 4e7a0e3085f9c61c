"""A paged 4-bit KV cache on the host: the quantiser's steps in fp32, attention in 64 bits, and the page tables as the header describes them, one
sequence after the other.  The tests of include/ckb200_cache.h hold the kernels to it."""
from __future__ import annotations

import numpy as np

BLOCK = 20


def quantize(x: np.ndarray) -> np.ndarray:
    """fp32 [..., 32 n] -> uint8 [..., 20 n]."""
    x = np.ascontiguousarray(x, dtype=np.float32).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(x).all(-1)
        low, high = x.min(-1), x.max(-1)
        m, d = low.astype(np.float16), ((high - low) / np.float32(15)).astype(np.float16)
        bad |= ~np.isfinite(m) | ~np.isfinite(d)
        step = d.astype(np.float32)
        inverse = np.where(step > 0, np.float32(1) / np.where(step > 0, step, np.float32(1)), np.float32(0))
        code = np.floor((x - m.astype(np.float32)[..., None]) * inverse[..., None] + np.float32(0.5))
        code = np.where(bad[..., None], 0, np.clip(np.nan_to_num(code), 0, 15)).astype(np.uint8)
    dm = np.stack([d, m], -1).view(np.uint16)
    dm[bad] = 0x7fff
    return np.concatenate([dm.view(np.uint8), code[..., :16] | code[..., 16:] << 4], -1).reshape(*x.shape[:-2], -1)


def values(rows: np.ndarray, dtype=np.float64) -> np.ndarray:
    """uint8 [..., 20 n] -> [..., 32 n]."""
    r = np.ascontiguousarray(rows).reshape(*rows.shape[:-1], -1, BLOCK)
    dm = np.ascontiguousarray(r[..., :4]).view(np.float16).astype(dtype)
    code = np.concatenate([r[..., 4:] & 15, r[..., 4:] >> 4], -1).astype(dtype)
    return (code * dm[..., :1] + dm[..., 1:]).reshape(*rows.shape[:-1], -1)


def magnitudes(rows: np.ndarray) -> np.ndarray:
    """|d| code + |m|: what rounding errors of a product with the row are proportional to."""
    r = np.ascontiguousarray(rows).reshape(*rows.shape[:-1], -1, BLOCK)
    dm = np.abs(np.ascontiguousarray(r[..., :4]).view(np.float16).astype(np.float64))
    code = np.concatenate([r[..., 4:] & 15, r[..., 4:] >> 4], -1).astype(np.float64)
    return (code * dm[..., :1] + dm[..., 1:]).reshape(*rows.shape[:-1], -1)


class Cache:
    """Pools [pages][kv heads][page_tokens][bytes] of K and V, a table and lengths."""

    def __init__(self, kv_heads, head_dim, page_tokens, pages, table, lens):
        self.kv_heads, self.head_dim, self.page_tokens, self.pages = kv_heads, head_dim, page_tokens, pages
        self.table, self.lens = np.array(table, dtype=np.int32), np.array(lens, dtype=np.int32)
        self.k = np.full((pages, kv_heads, page_tokens, head_dim // 32 * BLOCK), 255, dtype=np.uint8)      # d = m = NaN
        self.v = self.k.copy()

    def length(self, b):
        return int(np.clip(self.lens[b], 0, self.table.shape[1] * self.page_tokens))

    def place(self, b, pos):
        """(page, slot) of a position, None without one."""
        if pos < 0 or pos // self.page_tokens >= self.table.shape[1]:
            return None
        page = int(self.table[b, pos // self.page_tokens])
        return (page, pos % self.page_tokens) if 0 <= page < self.pages else None

    def store(self, k, v, tokens):
        """k, v: [batch * tokens][kv_heads * head_dim]."""
        for b in range(len(self.lens)):
            for t in range(tokens):
                at = self.place(b, self.length(b) - tokens + t)
                if at is None:
                    continue
                for pool, x in ((self.k, k), (self.v, v)):
                    pool[at[0], :, at[1]] = quantize(x[b * tokens + t].reshape(self.kv_heads, self.head_dim))

    def rows(self, b, keys, pool):
        """[kv heads][len(keys)][bytes] of positions that have a page."""
        at = [self.place(b, int(p)) for p in keys]
        return np.stack([pool[p, :, s] for p, s in at], 1)

    def attention(self, q, tokens, heads, window=0):
        """q [batch * tokens][heads * head_dim] -> (results in 64 bits, bound of the error of an fp32 computation) of the same shape.

        The bound: a score is a sum of head_dim products, each rounded and added in fp32, over terms of size |q| (|d| code + |m|); the
        kernels may also cut q to 22 bits (two fp16 pieces).  A score that is off by e makes its weight off by e, the sum of n weights by e
        and n roundings, and the result by twice that, times the largest value that it can be made of; 2^-20 for the exponential (two
        units in the last place), the scaling and the pieces of the weights."""
        hd, group = self.head_dim, heads // self.kv_heads
        out, off = np.zeros((len(q), heads, hd)), np.zeros((len(q), heads, hd))
        for b in range(len(self.lens)):
            for t in range(tokens):
                pos = self.length(b) - tokens + t
                keys = [p for p in range(max(0, pos - window + 1) if window else 0, pos + 1) if self.place(b, p)]
                if not keys:
                    continue
                rk, rv = self.rows(b, keys, self.k), self.rows(b, keys, self.v)
                k, v, ka, va = values(rk), values(rv), magnitudes(rk), magnitudes(rv)
                x = q[b * tokens + t].astype(np.float64).reshape(self.kv_heads, group, hd)
                s = np.einsum("hgd,hnd->hgn", x, k) / np.sqrt(hd)
                with np.errstate(all="ignore"):
                    w = np.exp(s - s.max(-1, keepdims=True))
                    o = np.einsum("hgn,hnd->hgd", w, v) / w.sum(-1, keepdims=True)
                size = (np.einsum("hgd,hnd->hgn", np.abs(x), ka) / np.sqrt(hd)).max(-1, keepdims=True)
                e = size * (hd * 2.0 ** -24 + 2.0 ** -21)
                out[b * tokens + t] = o.reshape(heads, hd)
                off[b * tokens + t] = (2 * (e + len(keys) * 2.0 ** -24) + 2.0 ** -20).repeat(hd, -1).reshape(heads, hd) * va.max(1)[:, None].repeat(group, 1).reshape(heads, hd)
        return out.reshape(len(q), -1), off.reshape(len(q), -1)

    def attention_weighed(self, q, tokens, heads, window=0):
        """As attention, with a bound in which every key counts by its weight and each channel by its own block.

        With z = |m| + 16 |d| for a block (the two terms d (code - 8) and m + 8 d that a value is made of are smaller together), w the weights relative to the largest and l
        their sum: a score that is off by e (the bound above) changes the result by w e (z + Z) / l, Z the mean of z; so do n roundings of the sums, and 2^-20 for the exponential,
        the scaling and the two fp16 pieces of weights, steps and middles, 22 bits each.  What is lost whatever the weight: a weight's pieces end at 2^-25 where the largest is 2^10 or
        more, 2^-35 z; the product of weight and step, rounded to two pieces that end at 2^-25 each, where the step is 2^-10 or more: 8 * 2^-24 / 2^10 * 2^10 |d| = 2^-21 |d|, or less than
        2^-32 z where the step is smaller than that, but z among the largest."""
        hd, group = self.head_dim, heads // self.kv_heads
        out, off = np.zeros((len(q), heads, hd)), np.zeros((len(q), heads, hd))
        for b in range(len(self.lens)):
            for t in range(tokens):
                pos = self.length(b) - tokens + t
                keys = [p for p in range(max(0, pos - window + 1) if window else 0, pos + 1) if self.place(b, p)]
                if not keys:
                    continue
                rk, rv = self.rows(b, keys, self.k), self.rows(b, keys, self.v)
                k, v, ka = values(rk), values(rv), magnitudes(rk)
                dm = np.abs(np.ascontiguousarray(rv.reshape(*rv.shape[:-1], -1, BLOCK)[..., :4]).view(np.float16).astype(np.float64)).repeat(32, -2)
                d, z = dm[..., 0], dm[..., 1] + 16 * dm[..., 0]
                x = q[b * tokens + t].astype(np.float64).reshape(self.kv_heads, group, hd)
                s = np.einsum("hgd,hnd->hgn", x, k) / np.sqrt(hd)
                w = np.exp(s - s.max(-1, keepdims=True))
                total = w.sum(-1, keepdims=True)
                e = np.einsum("hgd,hnd->hgn", np.abs(x), ka) / np.sqrt(hd) * (hd * 2.0 ** -24 + 2.0 ** -21)
                rel = w * (2 * e + 2 * len(keys) * 2.0 ** -24 + 2.0 ** -20)
                mean = np.einsum("hgn,hnd->hgd", w, z) / total
                out[b * tokens + t] = (np.einsum("hgn,hnd->hgd", w, v) / total).reshape(heads, hd)
                off[b * tokens + t] = ((np.einsum("hgn,hnd->hgd", rel, z) + rel.sum(-1, keepdims=True) * mean + (2.0 ** -21 * d + 2.0 ** -32 * z).sum(1)[:, None]) / total).reshape(heads, hd)
        return out.reshape(len(q), -1), off.reshape(len(q), -1)


class Tables:
    """Page tables, lengths and reference counts under the calls of the header; `pool` [planes][pages] is any array of page contents."""

    def __init__(self, batch, stride, pages, page_tokens, pool):
        self.table = np.full((batch, stride), -1, dtype=np.int32)
        self.lens, self.refs = np.zeros(batch, dtype=np.int32), np.zeros(pages, dtype=np.int32)
        self.pt, self.pool = page_tokens, pool

    def columns(self, n):
        return -(-int(n) // self.pt)

    def resize(self, new_lens):
        status = np.zeros(len(self.lens), dtype=np.int32)
        stride = self.table.shape[1]
        for b, n in enumerate(new_lens):
            if 0 <= n < self.lens[b]:
                for c in range(self.columns(n), self.columns(self.lens[b])):
                    if self.table[b, c] >= 0:
                        self.refs[self.table[b, c]] -= 1
                    self.table[b, c] = -1
                self.lens[b] = n
        for b, n in enumerate(new_lens):
            if n > stride * self.pt:
                status[b] = 1
                continue
            if n <= self.lens[b]:
                continue
            have, need = self.columns(self.lens[b]), self.columns(n)
            last = self.table[b, have - 1] if self.lens[b] % self.pt else -1
            copy = last >= 0 and self.refs[last] > 1
            free = np.flatnonzero(self.refs == 0)
            if len(free) < need - have + copy:
                status[b] = 1
                continue
            if copy:
                self.refs[last] -= 1
                self.pool[:, free[0]] = self.pool[:, last]
                self.table[b, have - 1] = free[0]
                self.refs[free[0]] = 1
                free = free[1:]
            self.table[b, have:need] = free[:need - have]
            self.refs[free[:need - have]] = 1
            self.lens[b] = n
        return status

    def fork(self, parent):
        table, lens = self.table.copy(), self.lens.copy()
        for b, p in enumerate(parent):
            if not 0 <= p < len(lens) or p == b:
                continue
            self.table[b], self.lens[b] = table[p], lens[p]
            for rows, by in ((table[p], 1), (table[b], -1)):
                for e in rows[rows >= 0]:
                    self.refs[e] += by

    def compact(self):
        used = np.flatnonzero(self.refs > 0)
        live = len(used)
        src, dst = used[used >= live], np.flatnonzero(self.refs[:live] == 0)
        for s, d in zip(src, dst):
            self.pool[:, d] = self.pool[:, s]
            self.refs[d], self.refs[s] = self.refs[s], 0
            self.table[self.table == s] = d
        return live
