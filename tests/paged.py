"""Paged KV caches for the tests: pages packed and read on the host, and the append
and the attention restated in 64 bits from their definitions."""
from __future__ import annotations

import numpy as np

from zlm_amd import device as zd


def round_scale(x):
    """x (float64) to the scale of a q4_0 block: 8 significant bits, an f16, at most 2720 in size."""
    f = np.asarray(x, np.float32)
    u = f.view(np.uint32).astype(np.uint64)
    u = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32)
    return np.clip(u.view(np.float32), -2720, 2720).astype(np.float16)


def quantise(x):
    """(nibbles, scales) of x [..., hd] (float64) in blocks of 32."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    at = np.argmax(np.where(np.isnan(b), -1.0, np.abs(b)), -1)[..., None]
    m = np.take_along_axis(b, at, -1)[..., 0]
    with np.errstate(invalid="ignore", divide="ignore"):
        d = round_scale(-m / 8)
        dd = d.astype(np.float64)[..., None]
        n = np.where(dd != 0, np.floor(b / np.where(dd != 0, dd, 1.0) + 8.5), 8.0)
    n = np.clip(np.nan_to_num(n, nan=0.0), 0, 15).astype(np.uint8)
    d = np.where(np.isnan(b).any(-1), np.float16(np.nan), d)
    return n.reshape(x.shape), d


class Pool:
    """K and V pools on the host, bytes [pages, kv, page * row bytes] each."""

    def __init__(self, kind, n_kv, hd, page, n_pages, fill=None):
        self.kind, self.n_kv, self.hd, self.page, self.n_pages = kind, n_kv, hd, page, n_pages
        self.row = 2 * hd if kind == zd.F16 else hd // 2 + hd // 16
        shape = (n_pages, n_kv, page * self.row)
        assert zd.paged_page_bytes(kind, n_kv, hd, page) == n_kv * page * self.row
        if fill is None:  # every bit set: NaN wherever a value is read that nobody wrote
            self.k, self.v = np.full(shape, 255, np.uint8), np.full(shape, 255, np.uint8)
        else:
            self.k, self.v = (fill.integers(0, 256, shape, dtype=np.uint8) for _ in range(2))

    def _k_parts(self):
        cut = self.page * self.hd // 2
        return (self.k[:, :, :cut].reshape(self.n_pages, self.n_kv, self.page, self.hd // 32, 16),
                self.k[:, :, cut:].view(np.float16).reshape(self.n_pages, self.n_kv, self.page, self.hd // 32))

    def _v_parts(self):
        cut = self.page * self.hd // 2
        return (self.v[:, :, :cut].view(np.uint32).reshape(self.n_pages, self.n_kv, self.page // 8, self.hd),
                self.v[:, :, cut:].view(np.float16).reshape(self.n_pages, self.n_kv, self.page // 8, self.hd // 32, 8))

    def write(self, page, off, k, v):
        """K and V (float64 [kv, hd]) of one position."""
        g, j = divmod(off, 8)
        if self.kind == zd.F16:
            with np.errstate(over="ignore"):
                self.k.view(np.float16).reshape(self.n_pages, self.n_kv, self.page, self.hd)[page, :, off] = k
                self.v.view(np.float16).reshape(self.n_pages, self.n_kv, self.page // 8, self.hd, 8)[page, :, g, :, j] = v
            return
        (kn, kd), (vn, vd) = quantise(k), quantise(v)
        self.put(page, off, kn, kd, vn, vd)

    def put(self, page, off, kn, kd, vn, vd):
        g, j = divmod(off, 8)
        cut = self.page * self.hd // 2
        b = kn.reshape(self.n_kv, self.hd // 32, 2, 16)
        row = slice(off * self.hd // 2, (off + 1) * self.hd // 2)
        self.k[page, :, :cut][:, row] = (b[:, :, 0] | (b[:, :, 1] << 4)).reshape(self.n_kv, -1)
        sc = self.k[page, :, cut:].view(np.float16)
        sc[:, off * self.hd // 32:(off + 1) * self.hd // 32] = kd
        sh = np.uint32(4 * (j // 2) + 16 * (j % 2))
        w = self.v[page, :, :cut].view(np.uint32)[:, g * self.hd:(g + 1) * self.hd]
        w[:] = (w & ~(np.uint32(15) << sh)) | (vn.astype(np.uint32) << sh)
        sc = self.v[page, :, cut:].view(np.float16).reshape(self.n_kv, self.page // 8, self.hd // 32, 8)
        sc[:, g, :, j] = vd

    def rows(self, pages, offs):
        """(K, V) float64 [n, kv, hd] of positions by page and offset."""
        g, j = offs // 8, offs % 8
        if self.kind == zd.F16:
            k = self.k.view(np.float16).reshape(self.n_pages, self.n_kv, self.page, self.hd)[pages, :, offs]
            v = self.v.view(np.float16).reshape(self.n_pages, self.n_kv, self.page // 8, self.hd, 8)[pages, :, g, :, j]
            return k.astype(np.float64), v.astype(np.float64)
        kb, kd = self._k_parts()
        kb = kb[pages, :, offs]
        k = (np.concatenate([kb & 15, kb >> 4], -1).astype(np.float64) - 8) * kd[pages, :, offs].astype(np.float64)[..., None]
        vw, vd = self._v_parts()
        sh = (4 * (j // 2) + 16 * (j % 2)).astype(np.uint32)[:, None, None]
        n = ((vw[pages, :, g] >> sh) & 15).astype(np.float64).reshape(len(pages), self.n_kv, -1, 32)
        v = (n - 8) * vd[pages, :, g, :, j].astype(np.float64)[..., None]
        return k.reshape(len(pages), self.n_kv, self.hd), v.reshape(len(pages), self.n_kv, self.hd)


class Batch:
    """Sequences of (rows, positions with them), their pages scattered over the pool."""

    def __init__(self, lens, page, rng, behind=0, spare=1, shared=0):
        self.lens, self.page = lens, page
        self.q_start = np.cumsum([0] + [n for n, _ in lens]).astype(np.int32)
        self.kv_len = np.array([e for _, e in lens], np.int32)
        self.n_tokens = int(self.q_start[-1]) + behind
        need = [max(0, -(-e // page)) for _, e in lens]
        self.n_pages = sum(need) + spare
        self.stride = max(need + [1]) + 1
        order = rng.permutation(self.n_pages).astype(np.int32)
        # what no position needs is no page number
        self.table = rng.choice(np.array([-1, -7, 1 << 30, self.n_pages], np.int32), (len(lens), self.stride))
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n

    def places(self):
        """(row, sequence, position) of every row."""
        for s, (n, end) in enumerate(self.lens):
            for i in range(n):
                yield int(self.q_start[s]) + i, s, end - n + i

    def spot(self, s, p):
        return int(self.table[s, p // self.page]), p % self.page


def fill(pool, batch, rng, std=1.0):
    """Random K and V in every position of the batch's sequences."""
    for s, (_, end) in enumerate(batch.lens):
        for p in range(end):
            page, off = batch.spot(s, p)
            if pool.kind == zd.F16:
                pool.write(page, off, *(std * rng.standard_normal((2, pool.n_kv, pool.hd))))
            else:
                kn, vn = rng.integers(0, 16, (2, pool.n_kv, pool.hd)).astype(np.uint8)
                kd, vd = round_scale(0.25 * std * rng.standard_normal((2, pool.n_kv, pool.hd // 32)))
                pool.put(page, off, kn, kd, vn, vd)


def rotate(x, base, pos):
    half = x.shape[-1] // 2
    a = pos * np.exp(np.arange(half) * (-2.0 / x.shape[-1]) * np.log(np.float64(np.float32(base))))
    c, s = np.cos(a), np.sin(a)
    return np.concatenate([x[..., :half] * c - x[..., half:] * s, x[..., :half] * s + x[..., half:] * c], -1)


def append(pool, batch, qkv, n_heads, eps, base, qn=None, kn=None):
    """q_out (float64, rows of no sequence NaN); writes K and V into the pool."""
    hd, kv = pool.hd, pool.n_kv
    out = np.full((batch.n_tokens, n_heads, hd), np.nan)
    for row, s, p in batch.places():
        x = qkv[row, :(n_heads + 2 * kv) * hd].astype(np.float64).reshape(-1, hd)
        q, k, v = x[:n_heads], x[n_heads:n_heads + kv], x[n_heads + kv:n_heads + 2 * kv]
        if p < 0:
            out[row] = 0
            continue
        if qn is not None:
            q = q / np.sqrt((q * q).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * qn.astype(np.float64)
            k = k / np.sqrt((k * k).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * kn.astype(np.float64)
        out[row] = rotate(q, base, p)
        if p // batch.page < batch.stride and 0 <= batch.table[s, p // batch.page] < pool.n_pages:
            page, off = batch.spot(s, p)
            pool.write(page, off, rotate(k, base, p), v)
    return out


def attend(pool, batch, q, n_heads, scale, window=0):
    """(out, bound) float64: the attention of every row (rows of no sequence NaN), and per row a bound of the
    kernel's distance from it.

    The bound: a score's error is at most A (2^-22 + 2 hd 2^-24) with A = scale * sum |q k| (the two f16 parts of
    q leave 2^-22 of it, every one of the 2 hd products' sums rounds once); that, the 2^-20 of exp2 and of the
    parts of a probability, and the roundings of n/32 + 64 sums each move a weight by that share of itself, and
    the result by at most twice that times the largest |v|; plus the weights under f16's smallest part, 2^-30 each."""
    hd, g = pool.hd, n_heads // pool.n_kv
    out = np.full((batch.n_tokens, n_heads, hd), np.nan)
    bound = np.zeros(batch.n_tokens)
    for row, s, p in batch.places():
        lo = max(0, p - window + 1) if window else 0
        at = np.arange(lo, p + 1)
        out[row] = 0
        if p < 0:
            continue
        pages = batch.table[s, at // batch.page]
        if ((pages < 0) | (pages >= pool.n_pages)).any():
            out[row] = np.nan
            continue
        k, v = pool.rows(pages, at % batch.page)
        for h in range(n_heads):
            x = k[:, h // g] * q[row, h].astype(np.float64)
            sc = x.sum(-1) * scale
            a = (np.abs(x).sum(-1) * abs(scale)).max()
            w = np.exp(sc - sc.max())
            out[row, h] = (w / w.sum()) @ v[:, h // g]
            n = len(at)
            e = a * (2.0 ** -22 + 2 * hd * 2.0 ** -24) + 2.0 ** -20 + (n / 32 + 64) * 2.0 ** -24 + n * 2.0 ** -30
            bound[row] = max(bound[row], 2 * e * np.abs(v[:, h // g]).max())
    return out, bound
