"""The paged KV cache on the GPU against its 64-bit restatement (tests/paged.py):
the append's bytes, the rows read back and the attention, over cache types, head
sizes, page sizes, groups, ragged lengths, padding, windows and missing pages.
Everything a call must not use holds NaN or no page number."""
import sys

import numpy as np
import pytest

from tests import paged
from zlm_amd import device as zd

pytestmark = pytest.mark.gpu

EPS, BASE = 1e-6, 1e6
TYPES = [zd.F16, zd.Q4_0]


def _say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


class _Box:
    """Device copies of a pool, a batch and what else a call takes."""

    def __init__(self, dev):
        self.dev, self.bufs = dev, []

    def up(self, a):
        a = np.ascontiguousarray(a)
        p = self.dev.dev_malloc(max(16, a.nbytes))
        self.bufs.append(p)
        if a.nbytes:
            self.dev.dev_upload(p, a)
        return p

    def down(self, p, like):
        out = np.empty_like(like)
        if out.nbytes:
            self.dev.dev_download(out, p)
        return out

    def cache(self, pool):
        self.k, self.v = self.up(pool.k), self.up(pool.v)
        return zd.PagedCache(self.k, self.v, pool.kind, pool.n_kv, pool.hd, pool.page, pool.n_pages)

    def batch(self, b):
        self.q_start, self.kv_len, self.table = self.up(b.q_start), self.up(b.kv_len), self.up(b.table)
        return zd.PagedBatch(len(b.lens), b.n_tokens, self.q_start, self.kv_len, self.table, b.stride)

    def free(self):
        self.dev.sync()
        for p in self.bufs:
            self.dev.dev_free(p)


@pytest.fixture
def box(dev):
    b = _Box(dev)
    yield b
    b.free()


# rows and positions of the sequences of a batch: single tokens, groups of 8 begun and ended in the middle, page
# borders, empty sequences, padding rows, far positions
APPENDS = [
    [(1, 1)],
    [(1, 17), (1, 8), (0, 5), (1, 64), (1, 100001)],
    [(3, 3), (9, 20), (0, 0), (16, 16), (5, 2), (2, 0), (1, 33)],
    [(70, 131), (33, 33)],
]


def _far(lens, page):
    """A batch whose early pages are absent: positions far into a sequence with a small pool."""
    return any(e > 10000 for _, e in lens)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd,page,kv,group", [(128, 64, 2, 4), (64, 16, 3, 1), (256, 32, 1, 5), (128, 256, 8, 2)])
@pytest.mark.parametrize("case", range(len(APPENDS)))
@pytest.mark.parametrize("norm", [True, False])
def test_append_and_read(box, kind, hd, page, kv, group, case, norm):
    lens = APPENDS[case]
    _say(f"append kind={kind} hd={hd} page={page} kv={kv} group={group} case={case} norm={norm}")
    rng = np.random.default_rng(case * 31 + hd + page)
    heads = kv * group
    b = paged.Batch(lens, page, rng, behind=3)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages, fill=rng)
    stride = (heads + 2 * kv) * hd + (5 if case == 2 else 0)
    qkv = (2 * rng.standard_normal((b.n_tokens, stride))).astype(np.float32)
    qkv[:, -32:] *= 1e-6  # V blocks of tiny values
    if case == 1:
        qkv[0, -64:-32] = 0  # and of none
    qn, kn = (1 + 0.1 * rng.standard_normal((2, hd))).astype(np.float32)
    q0 = np.full((b.n_tokens, heads, hd), 7.0, np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_qkv, d_q, d_qn, d_kn = box.up(qkv), box.up(q0), box.up(qn), box.up(kn)
    ok = box.dev.paged_append_enqueue(cache, batch, d_qkv, d_q, heads, EPS, BASE, q_norm_w=d_qn if norm else 0,
                                      k_norm_w=d_kn if norm else 0, qkv_stride=stride if case == 2 else 0)
    assert ok, box.dev.last_error()
    q = box.down(d_q, q0).astype(np.float64)
    k, v = box.down(box.k, pool.k), box.down(box.v, pool.v)
    want = paged.append(pool, b, qkv, heads, EPS, BASE, qn if norm else None, kn if norm else None)
    rows = ~np.isnan(want)
    # one rounding to f32; an angle of 1e5 in 64 bits is good to 1e5 2^-52
    np.testing.assert_allclose(q[rows], want[rows], rtol=2.0 ** -23, atol=1e-9)
    assert (q[~rows] == 7.0).all()
    np.testing.assert_array_equal(k, pool.k)
    np.testing.assert_array_equal(v, pool.v)
    # the rows read back
    k0 = np.full((b.n_tokens, kv, hd), 7.0, np.float32)
    d_k, d_v = box.up(k0), box.up(k0)
    assert box.dev.paged_read_enqueue(cache, batch, d_k, d_v), box.dev.last_error()
    gk, gv = box.down(d_k, k0), box.down(d_v, k0)
    wk, wv = k0.copy(), k0.copy()
    for row, s, p in b.places():
        wk[row] = wv[row] = 0
        if p >= 0:
            page_id, off = b.spot(s, p)
            wk[row], wv[row] = (x[0] for x in pool.rows(np.array([page_id]), np.array([off])))
    np.testing.assert_array_equal(gk, wk)
    np.testing.assert_array_equal(gv, wv)


@pytest.mark.parametrize("kind", TYPES)
def test_append_of_values_at_the_borders(box, kind):
    """NaN, infinities, the largest and the smallest values, and halves that round."""
    hd, kv, page = 128, 1, 16
    _say(f"append borders kind={kind}")
    rng = np.random.default_rng(5)
    b = paged.Batch([(9, 9)], page, rng)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages, fill=rng)
    qkv = rng.standard_normal((9, 3 * hd)).astype(np.float32)
    v = qkv[:, 2 * hd:]
    v[0, 3], v[1, 40] = np.nan, np.inf
    v[2, 70], v[3, :32] = -3e38, 1e-9
    v[4, :32] = np.where(np.arange(32) % 2, 8.0, -8.0)  # two of the largest size: the first decides
    v[5, :32] = np.arange(32) * 0.5 - 8
    v[6, :32] = 2.0 ** -24
    cache, batch = box.cache(pool), box.batch(b)
    d_qkv, d_q = box.up(qkv), box.up(np.zeros((9, hd), np.float32))
    assert box.dev.paged_append_enqueue(cache, batch, d_qkv, d_q, 1, EPS, BASE), box.dev.last_error()
    got = paged.Pool(kind, kv, hd, page, b.n_pages)
    got.k, got.v = box.down(box.k, pool.k), box.down(box.v, pool.v)
    paged.append(pool, b, qkv, 1, EPS, BASE)
    at = np.arange(9)
    pages = b.table[0, at // page]
    for g, w in zip(got.rows(pages, at % page), pool.rows(pages, at % page)):
        np.testing.assert_array_equal(g, w)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("pos", [0, 5, 90])
def test_largest_of_a_rotated_block(box, hd, pos):
    """Values of one size and both signs, which the rotation moves apart by less than 32 bits hold: the first of the
    largest in 64 bits gives the scale its sign."""
    kv, page = 2, 16
    _say(f"append ties hd={hd} pos={pos}")
    rng = np.random.default_rng(hd + pos)
    b = paged.Batch([(1, pos + 1)] * 4, page, rng)
    pool = paged.Pool(zd.Q4_0, kv, hd, page, b.n_pages, fill=rng)
    qkv = np.zeros((4, 1 + 2 * kv, hd), np.float32)
    qkv[:, 1:1 + kv, :hd // 2] = 8.0 * rng.choice([-1, 1], (4, kv, hd // 2))
    cache, batch = box.cache(pool), box.batch(b)
    d_qkv, d_q = box.up(qkv), box.up(np.zeros((4, hd), np.float32))
    assert box.dev.paged_append_enqueue(cache, batch, d_qkv, d_q, 1, EPS, BASE), box.dev.last_error()
    got = box.down(box.k, pool.k)
    paged.append(pool, b, qkv.reshape(4, -1), 1, EPS, BASE)
    np.testing.assert_array_equal(got, pool.k)


ATTENDS = [
    # (lens, window): one position, borders of the 32-position blocks, the 128-position units and of pages
    ([(1, 1)], 0),
    ([(1, 31), (1, 32), (1, 33), (0, 9), (1, 127), (1, 128), (1, 129)], 0),
    ([(1, 700), (1, 5), (1, 257)], 0),
    # a prompt from nothing, a chunk, a few tokens, padding rows, no rows
    ([(37, 37), (20, 150), (5, 300), (4, 2), (0, 0), (3, 0), (1, 64)], 0),
    ([(37, 37), (20, 150), (5, 300), (1, 900)], 1),
    ([(37, 37), (20, 150), (5, 300), (1, 900)], 50),
    ([(150, 400), (1, 3)], 128),
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd,page,kv,group", [(128, 64, 2, 4), (64, 16, 3, 1), (256, 32, 1, 5), (128, 16, 1, 8),
                                              (128, 256, 1, 33)])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention(box, kind, hd, page, kv, group, case):
    lens, window = ATTENDS[case]
    _say(f"attention kind={kind} hd={hd} page={page} kv={kv} group={group} case={case}")
    rng = np.random.default_rng(case * 17 + hd + group)
    heads = kv * group
    b = paged.Batch(lens, page, rng, behind=2)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    q = (1.5 * rng.standard_normal((b.n_tokens, heads, hd))).astype(np.float32)
    o0 = np.full_like(q, 7.0)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(o0)
    scale = hd ** -0.5
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, scale, window=window), box.dev.last_error()
    got = box.down(d_o, o0).astype(np.float64)
    want, bound = paged.attend(pool, b, q, heads, scale, window)
    rows = ~np.isnan(want)
    assert (got[~rows] == 7.0).all()  # rows behind the last sequence
    off = np.where(rows, np.abs(got - np.where(rows, want, 0)), 0).max((1, 2))
    assert (off <= bound).all(), (off.max(), bound[off.argmax()], int(off.argmax()))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lens", [[(1, 5000), (1, 1)], [(1, 9000)] * 3 + [(2, 300)] * 40])
def test_attention_over_many_shares(box, kind, lens):
    """Items longer than a workgroup's share, joined from several; and more items than shares end at."""
    hd, page, kv, group = 128, 64, 2, 4
    _say(f"attention shares kind={kind} {lens[0]}")
    rng = np.random.default_rng(len(lens))
    b = paged.Batch(lens, page, rng)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    heads = kv * group
    q = (3 * rng.standard_normal((b.n_tokens, heads, hd))).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(q)
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, hd ** -0.5), box.dev.last_error()
    got = box.down(d_o, q).astype(np.float64)
    want, bound = paged.attend(pool, b, q, heads, hd ** -0.5)
    off = np.abs(got - want).max((1, 2))
    assert (off <= bound).all(), (off.max(), bound[off.argmax()])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("route", paged.TWO_PARTS)
def test_both_parts_of_q_and_of_the_probabilities(box, kind, route):
    """Every route at the accuracy that 32-bit products have; one f16 part in place of two is off by more (shown for
    the oracle on the CPU)."""
    _say(f"attention parts kind={kind} {route}")
    x = paged.TwoParts(kind, **paged.TWO_PARTS[route])
    cache, batch = box.cache(x.pool), box.batch(x.batch)
    d_q, d_o = box.up(x.q), box.up(np.full_like(x.q, 7))
    assert box.dev.launch_log(True)
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, x.heads, float(x.scale), window=x.window), \
        box.dev.last_error()
    log = [(r["what"], r["block"]) for r in box.dev.launch_log_read()]
    box.dev.launch_log(False)
    names = [w for w, _ in log]
    assert ("paged attention of many rows" in names) == ("few" not in route)
    assert "merge" not in route or "paged attention of many rows, merge" in names
    if x.hd == 256 and "few" not in route:
        assert log[0][1] == (512 if "halved" in route else 256)
    got, want = box.down(d_o, x.q).astype(np.float64), x.want()
    assert (got[-1] == 7).all()
    assert np.abs(got[:-1] - want[:-1]).max() <= x.limit()


@pytest.mark.parametrize("kind", TYPES)
def test_missing_pages_poison_the_rows_that_see_them(box, kind):
    hd, page, kv, group = 64, 16, 2, 2
    _say(f"attention missing pages kind={kind}")
    rng = np.random.default_rng(3)
    # the second sequence lacks a page; the third's positions end behind its table; the window hides what the fourth lacks
    b = paged.Batch([(4, 60), (3, 60), (2, 40), (2, 200)], page, rng)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    b.table[1, 3] = b.n_pages
    b.table[3, :11] = -1
    b.lens[2] = (2, b.stride * page + 1)
    b.kv_len[2] = b.lens[2][1]
    heads = kv * group
    q = rng.standard_normal((b.n_tokens, heads, hd)).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(q)
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, 0.1, window=20), box.dev.last_error()
    got = box.down(d_o, q).astype(np.float64)
    assert np.isnan(got[4:9]).all()
    b.lens[2] = (2, 40)  # the oracle's rows of the other sequences
    want, bound = paged.attend(pool, b, q, heads, 0.1, 20)
    for rows in (slice(0, 4), slice(9, 11)):
        assert (np.abs(got[rows] - want[rows]).max((1, 2)) <= bound[rows]).all()


@pytest.mark.parametrize("kind", TYPES)
def test_scores_far_apart(box, kind):
    """Scores hundreds apart, rows whose maximum comes last, q of very different sizes, a q of zeros."""
    hd, page, kv, group = 128, 32, 1, 4
    _say(f"attention far scores kind={kind}")
    rng = np.random.default_rng(8)
    b = paged.Batch([(1, 600), (1, 77)], page, rng)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    q = rng.standard_normal((2, 4, hd)).astype(np.float32)
    q[0] *= np.array([60, 1e-12, 0, 1e4], np.float32)[:, None]
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(q)
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, 4, hd ** -0.5), box.dev.last_error()
    got = box.down(d_o, q).astype(np.float64)
    want, _ = paged.attend(pool, b, q, 4, hd ** -0.5)
    for h in range(4):
        sel = paged.attend(pool, b, np.where(np.arange(4)[None, :, None] == h, q, 0), 4, hd ** -0.5)[1]
        assert (np.abs(got[:, h] - want[:, h]).max(1) <= sel).all(), h


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-30])
@pytest.mark.parametrize("lens", [[(1, 200), (2, 9)], [(150, 200)]])
def test_other_scales(box, kind, scale, lens):
    """A scale of 0 (the mean of V), below 0 and so small that no score differs; few rows and many."""
    hd, page, kv, group = 64, 32, 1, 2
    _say(f"attention kind={kind} scale={scale} {lens}")
    rng = np.random.default_rng(31)
    b = paged.Batch(lens, page, rng)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    q = rng.standard_normal((b.n_tokens, kv * group, hd)).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(q)
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, kv * group, scale), box.dev.last_error()
    got = box.down(d_o, q)
    want, bound = paged.attend(pool, b, q, kv * group, np.float64(np.float32(scale)))
    assert (np.abs(got - want).max((1, 2)) <= bound).all()


class _Some:
    """A batch of which only some rows are looked at."""

    def __init__(self, b, rows):
        self.b, self.rows = b, rows

    def __getattr__(self, name):
        return getattr(self.b, name)

    def places(self):
        return (x for x in self.b.places() if x[0] in self.rows)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd,group,lens,window", [
    (256, 2, [(1100, 1300), (1, 9)], 0), (256, 2, [(1, 300), (1100, 1200)], 130), (256, 2, [(520, 600)], 0),
    (128, 4, [(2100, 2100), (3, 70)], 0), (64, 4, [(1100, 1111), (40, 40)], 0)])
def test_prompts_that_fill_the_chip(box, kind, hd, group, lens, window):
    """More tiles of rows than CUs, so that no positions are split, and just fewer; some of the rows are looked at."""
    page, kv = 32, 8
    _say(f"attention of prompts kind={kind} hd={hd} {lens} window={window}")
    rng = np.random.default_rng(35)
    b = paged.Batch(lens, page, rng, behind=1)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    heads = kv * group
    q = (1.5 * rng.standard_normal((b.n_tokens, heads, hd))).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(np.full_like(q, 7))
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, hd ** -0.5, window=window), box.dev.last_error()
    got = box.down(d_o, q)
    assert (got[-1] == 7).all()
    last = b.n_tokens - 2
    rows = sorted({0, 1, 15, 16, 31, 32, 63, 64, 500, 519, last - 1, last} | set(rng.integers(0, last, 12).tolist()))
    rows = [r for r in rows if r <= last]
    want, bound = paged.attend(pool, _Some(b, rows), q, heads, hd ** -0.5, window)
    assert (np.abs(got[rows] - want[rows]).max((1, 2)) <= bound[rows]).all()
    assert np.isfinite(got).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd,window", [(64, 0), (128, 0), (256, 33)])
@pytest.mark.parametrize("long", [60, 130])
def test_a_prompt_among_drafts(box, kind, hd, window, long):
    """Twenty sequences of a few tokens and one of many: with 60 tokens (8 heads, 792 rows) the few-row kernel takes
    the batch alone, or both do (f16, heads of 256); with 130 (1352 rows) both."""
    page, kv, group = 16, 1, 8
    _say(f"prompt among drafts kind={kind} hd={hd} long={long}")
    rng = np.random.default_rng(hd + long)
    lens = [(1 + i % 3, 9 + 7 * i) for i in range(20)]
    lens.insert(11, (long, long + 21))
    b = paged.Batch(lens, page, rng, behind=2)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    q = rng.standard_normal((b.n_tokens, kv * group, hd)).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(np.full_like(q, 7))
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, kv * group, hd ** -0.5, window=window), box.dev.last_error()
    got = box.down(d_o, q)
    want, bound = paged.attend(pool, b, q, kv * group, hd ** -0.5, window)
    assert (np.abs(got - want).max((1, 2))[:-2] <= bound[:-2]).all() and (got[-2:] == 7).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("live", [1, 8, 9, 32])
def test_one_sequence_of_fewer_rows(box, kind, hd, live):
    """One sequence that has a part of the token rows only: a prompt's last chunk in the buffers, or in the graph, of
    a full one (4 q heads: 4, 32, 36 and 128 rows of the attention's tiles)."""
    page, kv, group, most, kept = 32, 1, 4, 330, 45
    dev, heads = box.dev, kv * group
    _say(f"one sequence kind={kind} hd={hd} live={live}")
    rng = np.random.default_rng(hd + live)
    b = paged.Batch([(most, kept + most)], page, rng)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    q = rng.standard_normal((most, heads, hd)).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(np.full_like(q, 7))

    def step():
        assert dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, hd ** -0.5), dev.last_error()

    def check(lens, rows):
        b.lens = [lens]
        got = box.down(d_o, q)
        want, bound = paged.attend(pool, _Some(b, rows), q, heads, hd ** -0.5)
        assert (np.abs(got[rows] - want[rows]).max((1, 2)) <= bound[rows]).all()
        assert (got[lens[0]:] == 7).all()

    step()
    check((most, kept + most), [0, 17, most - 1])
    assert dev.capture_begin(), dev.last_error()
    step()
    g = dev.capture_end()
    assert g, dev.last_error()
    try:
        dev.dev_upload(box.q_start, np.array([0, live], np.int32))
        dev.dev_upload(box.kv_len, np.array([kept + live], np.int32))
        for run in (step, lambda: dev.graph_launch(g, 1), step):
            dev.dev_upload(d_o, np.full_like(q, 7))
            run()
            check((live, kept + live), list(range(live)))
    finally:
        dev.graph_destroy(g)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("long", [0, 40])
def test_the_largest_batch(box, kind, long):
    """1024 sequences of one token each, or with some of 40 tokens (f16: many rows) far behind the first."""
    hd, page, kv, group = 64, 16, 1, 4
    _say(f"attention of 1024 sequences kind={kind} long={long}")
    rng = np.random.default_rng(32)
    lens = [(1, 1 + i % 37) for i in range(1024)]
    if long:
        lens[300] = lens[1023] = (long, long + 5)
        lens[511] = (0, 3)
    b = paged.Batch(lens, page, rng, behind=1)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    q = rng.standard_normal((b.n_tokens, kv * group, hd)).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(np.full_like(q, 7))
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, kv * group, 0.2), box.dev.last_error()
    got = box.down(d_o, q)
    assert (got[-1] == 7).all()
    want, bound = paged.attend(pool, b, q, kv * group, np.float64(np.float32(0.2)))
    assert (np.abs(got - want).max((1, 2))[:-1] <= bound[:-1]).all()


@pytest.mark.parametrize("kind", TYPES)
def test_pages_past_32_bits(box, kind):
    """Pages that lie more than 2^32 bytes into the pools, few rows and many."""
    hd, page, kv, group = 256, 256, 8, 1
    _say(f"far pages kind={kind}")
    rng = np.random.default_rng(33)
    heads = kv * group
    b = paged.Batch([(1, 300), (200, 200)], page, rng, spare=0)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    page_bytes = zd.paged_page_bytes(kind, kv, hd, page)
    far = (1 << 32) // page_bytes + 7
    n_pages = far + b.n_pages
    k, v = (box.dev.dev_malloc(n_pages * page_bytes) for _ in range(2))
    box.bufs += [k, v]
    box.dev.dev_upload(k + far * page_bytes, pool.k)
    box.dev.dev_upload(v + far * page_bytes, pool.v)
    cache = zd.PagedCache(k, v, kind, kv, hd, page, n_pages)
    b.table = np.where((b.table >= 0) & (b.table < b.n_pages), b.table + far, -1).astype(np.int32)
    batch = box.batch(b)
    b.table = np.where(b.table >= 0, b.table - far, -1)  # the oracle's
    qkv = rng.standard_normal((b.n_tokens, (heads + 2 * kv) * hd)).astype(np.float32)
    like = np.zeros((b.n_tokens, heads, hd), np.float32)
    d_q, d_o = box.up(like), box.up(like)
    assert box.dev.paged_append_enqueue(cache, batch, box.up(qkv), d_q, heads, EPS, BASE), box.dev.last_error()
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, hd ** -0.5), box.dev.last_error()
    box.dev.dev_download(pool.k, k + far * page_bytes)
    box.dev.dev_download(pool.v, v + far * page_bytes)
    q, got = box.down(d_q, like), box.down(d_o, like)
    read = box.up(np.zeros((b.n_tokens, kv, hd), np.float32)), box.up(np.zeros((b.n_tokens, kv, hd), np.float32))
    assert box.dev.paged_read_enqueue(cache, batch, *read), box.dev.last_error()
    for row, s, p in b.places():
        page_id, off = b.spot(s, p)
        for buf, x in zip(read, pool.rows(np.array([page_id]), np.array([off]))):
            if row % 50 == 0:
                np.testing.assert_array_equal(box.down(buf, like[:, :kv])[row], x[0])
    few = [0, 1, 2, 77, 200]  # of the 201 rows
    want, bound = paged.attend(pool, _Some(b, few), q, heads, hd ** -0.5)
    assert (np.abs(got[few] - want[few]).max((1, 2)) <= bound[few]).all()
    ref = paged.append(paged.Pool(kind, kv, hd, page, b.n_pages), b, qkv, heads, EPS, BASE)
    np.testing.assert_allclose(q, ref, rtol=2.0 ** -23, atol=1e-9)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 40])
def test_last_positions(box, kind, hd, rows):
    """Windows that end at the last position a sequence can have, few rows and many (one page stands for all), and rows
    past it."""
    page, group, window, last = 256, 4, 40, (1 << 31) - 256
    _say(f"last positions kind={kind} hd={hd} rows={rows}")
    rng = np.random.default_rng(hd + rows)
    b = paged.Batch([(rows, page)], page, rng, spare=0)
    pool = paged.Pool(kind, 1, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    q = rng.standard_normal((rows, group, hd)).astype(np.float32)
    stride = (1 << 31) // page
    kv_len, d_q, d_o = box.up(np.array([last], np.int32)), box.up(q), box.up(np.full_like(q, 7))
    batch = zd.PagedBatch(1, rows, box.up(np.array([0, rows], np.int32)), kv_len, box.up(np.zeros((1, stride), np.int32)),
                          stride)
    cache = box.cache(pool)

    def run():
        assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, group, hd ** -0.5, window=window), \
            box.dev.last_error()
        return box.down(d_o, q)

    want, bound = paged.attend(pool, b, q, group, hd ** -0.5, window)
    assert (np.abs(run() - want).max((1, 2)) <= bound).all()
    for past in (1, 255):
        box.dev.dev_upload(kv_len, np.array([last + past], np.int32))
        got = run()
        assert np.isnan(got[max(0, rows - past):]).all() and np.isfinite(got[:max(0, rows - past)]).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("lens", [[(1, 100), (1, 90), (3, 40)], [(150, 200), (1, 150), (40, 120)]])
def test_sequences_that_share_pages(box, kind, lens):
    """A prefix that two sequences share, one page at two places of a table, few rows and many."""
    hd, page, kv, group = 128, 16, 1, 4
    _say(f"shared pages kind={kind} {lens}")
    rng = np.random.default_rng(36)
    b = paged.Batch(lens, page, rng)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    b.table[1:, :2] = b.table[0, :2]
    b.table[1, :4] = b.table[0, :4]
    b.table[2, 1] = b.table[2, 0]
    q = rng.standard_normal((b.n_tokens, kv * group, hd)).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(np.full_like(q, 7))
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, kv * group, hd ** -0.5), box.dev.last_error()
    got = box.down(d_o, q)
    want, bound = paged.attend(pool, b, q, kv * group, hd ** -0.5)
    assert (np.abs(got - want).max((1, 2)) <= bound).all()


def test_nan_in_one_sequence_stays_there(box):
    hd, page, kv, group = 128, 16, 1, 4
    rng = np.random.default_rng(9)
    b = paged.Batch([(1, 40), (1, 40)], page, rng)
    pool = paged.Pool(zd.F16, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    page_id, off = b.spot(0, 17)
    pool.write(page_id, off, np.full((kv, hd), np.nan), np.full((kv, hd), np.inf))
    q = rng.standard_normal((2, 4, hd)).astype(np.float32)
    q[1, 2, 5] = np.nan
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(q)
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, 4, hd ** -0.5), box.dev.last_error()
    got = box.down(d_o, q)
    assert np.isnan(got[0]).all() and np.isnan(got[1, 2]).all()
    assert np.isfinite(got[1, [0, 1, 3]]).all()


@pytest.mark.parametrize("kind", TYPES)
def test_captured_step_replays_for_later_lengths(box, kind):
    """Append and attention in a graph: replayed as the sequences grow, with eager work of another shape between,
    each replay against the eager calls; and a second graph over the same scratch."""
    hd, page, kv, group = 128, 16, 2, 4
    dev, heads = box.dev, kv * group
    _say(f"paged graph kind={kind}")
    rng = np.random.default_rng(12)
    b = paged.Batch([(1, 90), (1, 15), (1, 300)], page, rng)
    pool = paged.Pool(kind, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    qkv = rng.standard_normal((3, (heads + 2 * kv) * hd)).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_qkv, d_q, d_o = box.up(qkv), box.up(np.zeros((3, heads, hd), np.float32)), box.up(np.zeros((3, heads, hd), np.float32))
    d_o2 = box.up(np.zeros((3, heads, hd), np.float32))

    def step(out):
        assert dev.paged_append_enqueue(cache, batch, d_qkv, d_q, heads, EPS, BASE), dev.last_error()
        assert dev.paged_attention_enqueue(cache, batch, d_q, out, heads, hd ** -0.5), dev.last_error()

    step(d_o)
    graphs = []
    for out in (d_o, d_o2):
        assert dev.capture_begin(), dev.last_error()
        step(out)
        graphs.append(dev.capture_end())
        assert graphs[-1], dev.last_error()
    like = np.zeros((3, heads, hd), np.float32)
    try:
        for lens in ([90, 15, 300], [33, 14, 299], [81, 1, 64]):
            dev.dev_upload(box.kv_len, np.array(lens, np.int32))
            got = []
            for g, out in zip(graphs, (d_o, d_o2)):
                dev.dev_upload(d_o, np.full_like(like, 9))
                dev.graph_launch(g, 2)
                got.append(box.down(out, like))
                assert dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, 1.0, window=3), dev.last_error()
            dev.dev_upload(d_o, np.full_like(like, 9))
            step(d_o)
            want = box.down(d_o, like)
            assert np.isfinite(want).all()
            for x in got:
                np.testing.assert_array_equal(x, want)
    finally:
        for g in graphs:
            dev.graph_destroy(g)


def test_results_repeat(box):
    """The same call gives the same bits, whatever ran between."""
    hd, page, kv, group = 128, 64, 2, 4
    rng = np.random.default_rng(2)
    b = paged.Batch([(1, 2000), (6, 90), (1, 700)], page, rng)
    pool = paged.Pool(zd.Q4_0, kv, hd, page, b.n_pages)
    paged.fill(pool, b, rng)
    heads = kv * group
    q = rng.standard_normal((b.n_tokens, heads, hd)).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(q)
    got = []
    for _ in range(3):
        assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, 0.09), box.dev.last_error()
        got.append(box.down(d_o, q))
        assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, 0.5, window=7), box.dev.last_error()
    np.testing.assert_array_equal(got[0], got[1])
    np.testing.assert_array_equal(got[0], got[2])
