"""An e4m3 paged cache for the tests, and attention by a window beside sinks, restated in
64 bits from their definitions (the rest is tests/paged.py's)."""
from __future__ import annotations

import numpy as np

from tests import paged
from zlm_amd import device as zd

LEAST, MOST = 112, 134  # scale bytes


def _numbers():
    """The values of codes 0 to 127 (the last NaN)."""
    c = np.arange(128)
    e, m = c >> 3, c & 7
    v = np.where(e == 0, np.ldexp(m.astype(np.float64), -9), np.ldexp(8.0 + m, e - 10))
    v[127] = np.nan
    return v


NUMBERS = _numbers()


def decode(codes, byte):
    k = np.clip(byte.astype(np.int64), LEAST, MOST) - 127
    return np.where(codes >= 128, -1.0, 1.0) * NUMBERS[codes & 127] * np.ldexp(1.0, k)


def encode(x, byte):
    """Codes nearest to x (float64) at scale bytes (of LEAST to MOST; broadcast), halves to the even code."""
    y = np.clip(x, -57344, 57344) * np.ldexp(1.0, 127 - np.asarray(byte, np.int64))
    a = np.abs(y)
    hi = np.clip(np.searchsorted(NUMBERS[:127], a), 1, 126)
    below, above = a - NUMBERS[hi - 1], NUMBERS[hi] - a
    c = np.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, hi - 1)
    c = np.where(np.isnan(x), 127, c)
    return (c | np.where(np.signbit(x) & ~np.isnan(x), 128, 0)).astype(np.uint8)


def scale_byte(m):
    """Of blocks whose largest are m: the least k with m <= 448 2^k."""
    limits = 448 * np.ldexp(1.0, np.arange(LEAST - 127, MOST - 127))
    return LEAST + (np.asarray(m)[..., None] > limits).sum(-1)


class Pool:
    """K and V pools on the host, bytes [pages, kv, page * hd + 16] each, with the interface of paged.Pool.  write()
    keeps a position's values back until flush(), which is one append's."""

    kind = zd.CACHE_E4M3

    def __init__(self, n_kv, hd, page, n_pages, fill=None):
        self.n_kv, self.hd, self.page, self.n_pages, self.pending = n_kv, hd, page, n_pages, []
        shape = (n_pages, n_kv, page * hd + 16)
        assert zd.paged_page_bytes(self.kind, n_kv, hd, page) == n_kv * shape[2]
        if fill is None:
            self.k, self.v = np.full(shape, 255, np.uint8), np.full(shape, 255, np.uint8)
        else:  # any numbers, scale bytes also outside what is written
            self.k, self.v = (fill.integers(0, 256, shape, dtype=np.uint8) for _ in range(2))
            for p in (self.k, self.v):
                codes = p[:, :, :page * hd]
                codes[codes & 127 == 127] = 3
                p[:, :, page * hd:] = fill.integers(100, 140, shape[:2] + (16,), dtype=np.uint8)

    def parts(self, side):
        """(codes [pages, kv, page, hd], scale bytes [pages, kv, page / 16]), views of the pool."""
        n = self.page * self.hd
        p = getattr(self, side)
        codes = p[:, :, :n]
        if side == "k":
            codes = np.lib.stride_tricks.as_strided(codes, (self.n_pages, self.n_kv, self.page, self.hd),
                                                    codes.strides[:2] + (self.hd, 1))
        else:
            v = np.lib.stride_tricks.as_strided(codes, (self.n_pages, self.n_kv, self.page // 8, 8, self.hd),
                                                codes.strides[:2] + (8 * self.hd, 1, 8))
            return v, p[:, :, n:n + self.page // 16]
        return codes, p[:, :, n:n + self.page // 16]

    def _at(self, side, codes, page, off):
        return codes[page, :, off] if side == "k" else codes[page, :, off // 8, off % 8]

    def write(self, page, off, k, v):
        self.pending.append((page, off, np.array(k, np.float64), np.array(v, np.float64)))

    def flush(self):
        blocks = {}
        for page, off, k, v in self.pending:
            blocks.setdefault((page, off // 16), []).append((off, k, v))
        self.pending = []
        for (page, blk), rows in blocks.items():
            first = min(off for off, _, _ in rows)
            for i, side in enumerate("kv"):
                codes, scales = self.parts(side)
                x = np.stack([r[1 + i] for r in rows])
                with np.errstate(invalid="ignore"):
                    byte = scale_byte(np.nan_to_num(np.abs(x), nan=0.0, posinf=np.inf).max((0, 2)))
                if first % 16:
                    had = np.clip(scales[page, :, blk].astype(np.int64), LEAST, MOST)
                    byte = np.maximum(byte, had)
                    for off in range(16 * blk, first):
                        at = self._at(side, codes, page, off)
                        risen = (byte > had)[:, None]
                        at[...] = np.where(risen, encode(decode(at, had[:, None]), byte[:, None]), at)
                for off, *values in rows:
                    self._at(side, codes, page, off)[...] = encode(values[i], byte[:, None])
                scales[page, :, blk] = byte

    def rows(self, pages, offs):
        """(K, V) float64 [n, kv, hd] of positions by page and offset."""
        got = []
        for side in "kv":
            codes, scales = self.parts(side)
            c = codes[pages, :, offs] if side == "k" else codes[pages, :, offs // 8, offs % 8]
            got.append(decode(c, scales[pages, :, offs // 16][..., None]))
        return tuple(got)


def pool(kind, n_kv, hd, page, n_pages, fill=None):
    """A pool of any cache type."""
    if kind == zd.CACHE_E4M3:
        return Pool(n_kv, hd, page, n_pages, fill)
    return paged.Pool(kind, n_kv, hd, page, n_pages, fill)


def fill(p, batch, rng, std=1.0):
    """Random K and V in every position of the batch's sequences that has a page."""
    if p.kind != zd.CACHE_E4M3:
        paged.fill(p, batch, rng, std)
        return
    for s, (_, end) in enumerate(batch.lens):
        for pos in range(end):
            p.write(*batch.spot(s, pos), *(std * rng.standard_normal((2, p.n_kv, p.hd))))
    p.flush()


def append(p, batch, qkv, *args):
    q = paged.append(p, batch, qkv, *args)
    if p.kind == zd.CACHE_E4M3:
        p.flush()
    return q


def seen(p, window, sinks):
    """The positions that a row at p sees."""
    lo = max(0, p - window + 1) if window else 0
    return np.concatenate([np.arange(min(sinks, lo)), np.arange(lo, p + 1)])


def attend(pool, batch, q, n_heads, scale, window=0, sinks=0):
    """(out, bound) float64 as paged.attend has them, over the window and the sinks."""
    hd, g = pool.hd, n_heads // pool.n_kv
    out = np.full((batch.n_tokens, n_heads, hd), np.nan)
    bound = np.zeros(batch.n_tokens)
    for row, s, p in batch.places():
        out[row] = 0
        if p < 0:
            continue
        at = seen(p, window, sinks)
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


def as_e4m3(x):
    """A paged.TwoParts (made for an f16 cache) over an e4m3 one: its K and V are small whole numbers."""
    f16, b = x.pool, x.batch
    x.pool = Pool(f16.n_kv, f16.hd, f16.page, f16.n_pages)
    for s, (_, end) in enumerate(b.lens):
        for p in range(end):
            page, off = b.spot(s, p)
            k, v = f16.rows(np.array([page]), np.array([off]))
            x.pool.write(page, off, k[0], v[0])
    x.pool.flush()
    return x
