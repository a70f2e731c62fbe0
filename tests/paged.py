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


class TwoParts:
    """A case of the attention whose result is known to a few 1e-6, and is off by many times that where q or the
    probabilities enter a product as one f16 instead of two.

    K of position j is g(j) c with g = 1, 0, -1, 1, .. and c of ones and minus ones; q is a sign a dim plus 2^-12 c.
    So a row has three scores, 0 and plus and minus one number; every product and sum of q and K is exact in 32 bits;
    and what lies behind q's first 11 bits adds up: 2^-12 hd of a raw score of hd/4 at most.  V is u(g), whole numbers,
    so the parts of a probability that are lost add up too."""

    def __init__(self, kind, n_kv, hd, group, page, lens, window=0, seed=0):
        rng = np.random.default_rng(seed)
        self.heads, self.hd, self.window, self.scale = n_kv * group, hd, window, np.float32(5.2 / hd)
        self.batch = b = Batch(lens, page, rng, behind=1)
        self.pool = Pool(kind, n_kv, hd, page, b.n_pages)
        self.c = rng.choice([-1, 1], (n_kv, hd))
        self.u = rng.integers(-8, 8, (3, n_kv, hd))  # by g + 1
        self.u[:, :, 0] = [[-8], [7], [7]]  # two dims that show most of a weight
        self.u[:, :, 1] = [[7], [7], [-8]]
        one = np.ones((n_kv, hd // 32), np.float16)
        for s, (_, end) in enumerate(lens):
            for p in range(end):
                k, v = self.g(p) * self.c, self.u[self.g(p) + 1]
                spot = b.spot(s, p)
                if kind == zd.F16:
                    self.pool.write(*spot, k, v)
                else:
                    self.pool.put(*spot, (k + 8).astype(np.uint8), one, (v + 8).astype(np.uint8), one)
        # signs of q: half the dims like c's and up to an eighth more, or fewer
        m = hd // 2 + rng.integers(-(hd // 8), hd // 8 + 1, (b.n_tokens, self.heads))
        like = rng.permuted(np.broadcast_to(np.arange(hd), (b.n_tokens, self.heads, hd)), axis=-1) < m[..., None]
        c = np.repeat(self.c, group, 0)
        self.signs = np.where(like, c, -c)
        self.q = (self.signs + 2.0 ** -12 * c).astype(np.float32)
        assert (self.q == self.signs + 2.0 ** -12 * c).all()

    @staticmethod
    def g(p):
        return (p + 2) % 3 - 1  # 1, -1, 0, 1, ..

    def _rows(self):
        """(row, first and last position it sees) of the rows that see any."""
        at = [(r, max(0, p - self.window + 1) if self.window else 0, p) for r, _, p in self.batch.places() if p >= 0]
        return np.array(at).T

    def want(self, q_parts=2, p_parts=2):
        """The result in 64 bits (rows of no sequence NaN); with one part: what one f16 of q, or of the probabilities
        (scaled as the kernels scale them: 2^6 at the largest), makes of it."""
        out = np.full(self.q.shape, np.nan)
        row, lo, hi = self._rows()
        c = np.repeat(self.c, self.heads // len(self.c), 0)
        q = self.q.astype(np.float64) if q_parts == 2 else self.q.astype(np.float16).astype(np.float64)
        s = (q[row] * c).sum(-1) * np.float64(self.scale)  # of g = 1
        g = np.arange(-1, 2)
        seen = (self.g(np.arange(hi.max() + 1))[None] == g[:, None]).cumsum(1)
        n = seen[:, hi] - np.where(lo > 0, seen[:, lo - 1], 0)  # [3, rows]
        e = g[:, None, None] * s[None]
        top = np.where(n[:, :, None] > 0, e, -np.inf).max(0)
        w = np.exp(e - top) * 64
        first = w if p_parts == 2 else w.astype(np.float16).astype(np.float64)
        total = (n[:, :, None] * w).sum(0)
        u = np.repeat(self.u, self.heads // len(self.c), 1).astype(np.float64)
        out[row] = np.einsum("grh,ghd->rhd", n[:, :, None] * first, u) / total[..., None]
        return out

    def limit(self):
        """How far the kernels may be off.  In units of 2^-24, for exponents of two of A = 2.5 at most (1.3 of the raw
        score of hd/4 and its 2^-10, times log2 e, is 1.9): the factor of the scores is rounded twice (4 A), an
        exponent once (2 A + 6) and its base once (A + 6), three joins of sums round a difference of maxima (2 A each):
        times ln 2; exp2 and the joins' factors and products 2 + 3 x 3; the two parts of a probability leave 2^-20 (16).
        That is a weight's share; the result moves by twice it, and by the roundings of the sums, eight for every 32
        positions of a wave that takes them all and 64 for the rest, each once of the largest value, 8."""
        a = 2.5
        weight = np.log(2) * (4 * a + 2 * a + 6 + a + 6 + 3 * 2 * a) + 2 + 9 + 16
        _, lo, hi = self._rows()
        return 8 * 2.0 ** -24 * (2 * weight + (hi - lo + 1).max() / 4 + 64)


# One case a route of the attention: (heads, rows and positions, window)
TWO_PARTS = {
    "few": dict(n_kv=1, hd=128, group=4, page=64, lens=[(1, 300), (2, 90)]),
    "few, short": dict(n_kv=2, hd=64, group=8, page=16, lens=[(1, 30)] * 5),
    "few, heads of 256": dict(n_kv=2, hd=256, group=3, page=32, lens=[(1, 200), (1, 500)]),
    "many and merge, heads of 64": dict(n_kv=1, hd=64, group=4, page=32, lens=[(70, 700)]),
    "many and merge": dict(n_kv=1, hd=128, group=4, page=32, lens=[(70, 700)]),
    "halved and merge": dict(n_kv=1, hd=256, group=4, page=32, lens=[(70, 700)]),
    "many": dict(n_kv=8, hd=128, group=4, page=64, lens=[(2100, 2100)], window=100),
    "many, heads of 64": dict(n_kv=8, hd=64, group=8, page=64, lens=[(1050, 1050)], window=100),
    "many, heads of 256": dict(n_kv=8, hd=256, group=2, page=64, lens=[(1100, 1100)], window=100),
    "halved": dict(n_kv=8, hd=256, group=2, page=64, lens=[(520, 600), (1, 40)], window=100),
}
