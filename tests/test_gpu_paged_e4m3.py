"""The e4m3 paged cache on the GPU against its 64-bit restatement (tests/paged_more.py): the
append's bytes and scales, whole blocks, blocks begun and gone on with, the rows read back,
and the attention on every route.  What a call must not use holds NaN."""
import numpy as np
import pytest

from tests import paged, paged_more
from tests.test_gpu_paged import APPENDS, ATTENDS, BASE, EPS, _Box, _say, _Some
from zlm_amd import device as zd

pytestmark = pytest.mark.gpu

E4M3 = zd.CACHE_E4M3
SIZES = [(128, 64, 2, 4), (64, 16, 3, 1), (256, 32, 1, 5), (128, 256, 8, 2)]


@pytest.fixture
def box(dev):
    b = _Box(dev)
    yield b
    b.free()


def _same(got, pool, hd, page):
    """The pools' bytes (of scales only those that are blocks')."""
    for g, side in zip(got, "kv"):
        np.testing.assert_array_equal(g, getattr(pool, side), side)


@pytest.mark.parametrize("hd,page,kv,group", SIZES)
@pytest.mark.parametrize("case", range(len(APPENDS)))
@pytest.mark.parametrize("norm", [True, False])
def test_append_and_read(box, hd, page, kv, group, case, norm):
    lens = APPENDS[case]
    _say(f"append e4m3 hd={hd} page={page} kv={kv} group={group} case={case} norm={norm}")
    rng = np.random.default_rng(case * 37 + hd + page)
    heads = kv * group
    b = paged.Batch(lens, page, rng, behind=3)
    pool = paged_more.Pool(kv, hd, page, b.n_pages, fill=rng)
    stride = (heads + 2 * kv) * hd + (5 if case == 2 else 0)
    qkv = (2 * rng.standard_normal((b.n_tokens, stride))).astype(np.float32)
    qkv[:, -hd:] *= 1e-6  # the last head's V: tiny values
    if case == 1:
        qkv[0, -2 * hd:] = 0
    qn, kn = (1 + 0.1 * rng.standard_normal((2, hd))).astype(np.float32)
    q0 = np.full((b.n_tokens, heads, hd), 7.0, np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_qkv, d_q, d_qn, d_kn = box.up(qkv), box.up(q0), box.up(qn), box.up(kn)
    ok = box.dev.paged_append_enqueue(cache, batch, d_qkv, d_q, heads, EPS, BASE, q_norm_w=d_qn if norm else 0,
                                      k_norm_w=d_kn if norm else 0, qkv_stride=stride if case == 2 else 0)
    assert ok, box.dev.last_error()
    q = box.down(d_q, q0).astype(np.float64)
    got = box.down(box.k, pool.k), box.down(box.v, pool.v)
    want = paged_more.append(pool, b, qkv, heads, EPS, BASE, qn if norm else None, kn if norm else None)
    rows = ~np.isnan(want)
    np.testing.assert_allclose(q[rows], want[rows], rtol=2.0 ** -23, atol=1e-9)
    assert (q[~rows] == 7.0).all()
    _same(got, pool, hd, page)
    k0 = np.full((b.n_tokens, kv, hd), 7.0, np.float32)
    d_k, d_v = box.up(k0), box.up(k0)
    assert box.dev.paged_read_enqueue(cache, batch, d_k, d_v), box.dev.last_error()
    wk, wv = k0.copy(), k0.copy()
    for row, s, p in b.places():
        wk[row] = wv[row] = 0
        if p >= 0:
            page_id, off = b.spot(s, p)
            wk[row], wv[row] = (x[0] for x in pool.rows(np.array([page_id]), np.array([off])))
    np.testing.assert_array_equal(box.down(d_k, k0), wk)
    np.testing.assert_array_equal(box.down(d_v, k0), wv)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("steps", [(1,) * 35, (3, 1, 13, 2, 16, 5), (7, 40, 1, 1)])
def test_blocks_gone_on_with(box, hd, steps):
    """A sequence that grows by calls of a few rows each: values that rise by orders of magnitude within a block (so
    that its scale does), fall again, and rows of zeros."""
    page, kv, heads = 32, 2, 3
    _say(f"append e4m3 steps hd={hd} {steps}")
    rng = np.random.default_rng(hd + len(steps))
    n = sum(steps)
    b = paged.Batch([(n, n)], page, rng, behind=0)
    pool = paged_more.Pool(kv, hd, page, b.n_pages, fill=rng)
    qkv = rng.standard_normal((n, heads + 2 * kv, hd)).astype(np.float32)
    size = (10.0 ** rng.uniform(-5, 4, (n, 1, 1))).astype(np.float32)
    size[5] = 0
    qkv[:, heads:] *= size
    qkv = qkv.reshape(n, -1)
    cache, d_q = box.cache(pool), box.up(np.zeros((n, heads, hd), np.float32))
    at = 0
    for m in steps:
        b.lens, b.q_start, b.n_tokens = [(m, at + m)], np.array([0, m], np.int32), m
        b.kv_len = np.array([at + m], np.int32)
        batch = box.batch(b)
        rows = np.ascontiguousarray(qkv[at:at + m])
        assert box.dev.paged_append_enqueue(cache, batch, box.up(rows), d_q, heads, EPS, BASE), box.dev.last_error()
        paged_more.append(pool, b, rows, heads, EPS, BASE)
        box.k, box.v = cache.c.k, cache.c.v
        _same((box.down(box.k, pool.k), box.down(box.v, pool.v)), pool, hd, page)
        at += m


def test_values_at_the_borders(box):
    """NaN, infinities, the largest and smallest, halves that round to either side, and the borders of the scales."""
    hd, kv, page = 128, 1, 16
    _say("append e4m3 borders")
    rng = np.random.default_rng(5)
    lens = [(1, 1)] * 12
    b = paged.Batch(lens, page, rng)
    pool = paged_more.Pool(kv, hd, page, b.n_pages, fill=rng)
    qkv = rng.standard_normal((12, 3 * hd)).astype(np.float32)
    up = lambda x: np.nextafter(np.float32(x), np.float32(np.inf))  # noqa: E731
    for side in (1, 2):  # positions 0: K is not turned
        v = qkv[:, side * hd:(side + 1) * hd]
        v[0, 3] = np.nan
        v[1, 40] = np.inf
        v[2, 70] = -3e38
        v[3] = 1e-30
        v[4] = 0
        v[5, 0], v[6, 0], v[7, 0] = 448, up(448), -224
        v[8, :32] = 256 + 8 * np.arange(32)  # halves between numbers 32 apart, and at the border 448
        v[9, :] = 448 * 2.0 ** -rng.integers(0, 30, hd)
        v[10, 0] = up(57344)
        v[11, :] = np.nan
    cache, batch = box.cache(pool), box.batch(b)
    d_qkv, d_q = box.up(qkv), box.up(np.zeros((12, hd), np.float32))
    assert box.dev.paged_append_enqueue(cache, batch, d_qkv, d_q, 1, EPS, BASE), box.dev.last_error()
    got = paged_more.Pool(kv, hd, page, b.n_pages)
    got.k, got.v = box.down(box.k, pool.k), box.down(box.v, pool.v)
    paged_more.append(pool, b, qkv, 1, EPS, BASE)
    pages = b.table[:12, 0]
    for g, w in zip(got.rows(pages, np.zeros(12, int)), pool.rows(pages, np.zeros(12, int))):
        np.testing.assert_array_equal(g, w)
    for side in "kv":
        np.testing.assert_array_equal(got.parts(side)[1][pages], pool.parts(side)[1][pages])


@pytest.mark.parametrize("hd,page,kv,group", [(128, 64, 2, 4), (64, 16, 3, 1), (256, 32, 1, 5), (128, 16, 1, 8),
                                              (128, 256, 1, 33)])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention(box, hd, page, kv, group, case):
    lens, window = ATTENDS[case]
    _say(f"attention e4m3 hd={hd} page={page} kv={kv} group={group} case={case}")
    rng = np.random.default_rng(case * 19 + hd + group)
    heads = kv * group
    b = paged.Batch(lens, page, rng, behind=2)
    pool = paged_more.Pool(kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
    q = (1.5 * rng.standard_normal((b.n_tokens, heads, hd))).astype(np.float32)
    o0 = np.full_like(q, 7.0)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(o0)
    scale = hd ** -0.5
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, scale, window=window), box.dev.last_error()
    got = box.down(d_o, o0).astype(np.float64)
    want, bound = paged_more.attend(pool, b, q, heads, scale, window)
    rows = ~np.isnan(want)
    assert (got[~rows] == 7.0).all()
    off = np.where(rows, np.abs(got - np.where(rows, want, 0)), 0).max((1, 2))
    assert (off <= bound).all(), (off.max(), bound[off.argmax()], int(off.argmax()))


@pytest.mark.parametrize("route", paged.TWO_PARTS)
def test_both_parts_of_q_and_of_the_probabilities(box, route):
    _say(f"attention parts e4m3 {route}")
    x = paged_more.as_e4m3(paged.TwoParts(zd.F16, **paged.TWO_PARTS[route]))
    cache, batch = box.cache(x.pool), box.batch(x.batch)
    d_q, d_o = box.up(x.q), box.up(np.full_like(x.q, 7))
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, x.heads, float(x.scale), window=x.window), \
        box.dev.last_error()
    got, want = box.down(d_o, x.q).astype(np.float64), x.want()
    assert (got[-1] == 7).all()
    assert np.abs(got[:-1] - want[:-1]).max() <= x.limit()


@pytest.mark.parametrize("lens", [[(1, 40)], [(160, 160)]])
@pytest.mark.parametrize("std", [2.0 ** -16, 2.0 ** -21, 2e3])
def test_scales_at_both_ends(box, lens, std):
    """Blocks at the least and the largest scale: their values are f16's smallest, subnormal ones, and its largest.
    (Of weights that all count, so that V's values show; 2^-24 of V for what f16 leaves of P.)"""
    hd, page, kv, group = 128, 16, 1, 2
    _say(f"attention e4m3 ends {lens} std={std}")
    rng = np.random.default_rng(6)
    b = paged.Batch(lens, page, rng)
    pool = paged_more.Pool(kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng, std)
    codes, scales = pool.parts("v")
    used = scales[b.table[0, :-(-lens[0][1] // page)]]
    assert (used == (paged_more.LEAST if std < 1 else used)).all() and ((codes & 127) != 0).any()
    q = (rng.standard_normal((b.n_tokens, kv * group, hd)) / std).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(q)
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, kv * group, 0.01), box.dev.last_error()
    got = box.down(d_o, q)
    want, bound = paged_more.attend(pool, b, q, kv * group, np.float64(np.float32(0.01)))
    assert (np.abs(got - want).max((1, 2)) <= bound).all(), np.abs(got - want).max() / bound.max()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(1, 40)], [(160, 160)]])
@pytest.mark.parametrize("scales", [(134,), (135, 255), (112,), (0, 111)])
def test_scales_at_their_limits_and_past_them(box, hd, lens, scales):
    """Every block that is seen at the largest scale (K and V with 57344 and -57344 in each) or at the least one, or at
    a byte past these, which counts as them: the rows read back exactly, and the attention on both routes."""
    page, kv, group = 16, 2, 2
    _say(f"attention e4m3 limits hd={hd} {lens} scales={scales}")
    rng = np.random.default_rng(hd + scales[0])
    b = paged.Batch(lens, page, rng)
    pool = paged_more.Pool(kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
    used = b.table[0, :-(-lens[0][1] // page)]
    for side in "kv":
        codes, of_block = pool.parts(side)
        for i, page_id in enumerate(used):
            for h in range(kv):
                of_block[page_id, h, 0] = scales[(i + h) % len(scales)]
                for at, code in enumerate((126, 254)):  # 448, -448
                    off, dim = (0, int(rng.integers(hd))) if side == "k" else (at % page, int(rng.integers(hd)))
                    if side == "k":
                        codes[page_id, h, off, dim] = code
                    else:
                        codes[page_id, h, off // 8, off % 8, dim] = code
    offs = np.arange(lens[0][1])
    k, v = pool.rows(used[offs // page], offs % page)
    most = 57344 if scales[0] > 112 else 448 * 2.0 ** -15
    assert np.abs(k).max() == most and np.abs(v).max() == most and np.isfinite(k).all() and np.isfinite(v).all()
    q = (rng.standard_normal((b.n_tokens, kv * group, hd)) * (16 / most)).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    n = lens[0][0]
    like = np.zeros((n, kv, hd), np.float32)
    d_k, d_v = box.up(like), box.up(like)
    assert box.dev.paged_read_enqueue(cache, batch, d_k, d_v), box.dev.last_error()
    np.testing.assert_array_equal(box.down(d_k, like), k[-n:])
    np.testing.assert_array_equal(box.down(d_v, like), v[-n:])
    d_q, d_o = box.up(q), box.up(q)
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, kv * group, 0.01), box.dev.last_error()
    got = box.down(d_o, q)
    want, bound = paged_more.attend(pool, b, q, kv * group, np.float64(np.float32(0.01)))
    assert (np.abs(got - want).max((1, 2)) <= bound).all(), np.abs(got - want).max() / bound.max()
    assert bound.max() <= most * 2.0 ** -10  # (tight enough to tell a scale from the next)


@pytest.mark.parametrize("hd,group,lens,window", [
    (256, 2, [(1100, 1300), (1, 9)], 0), (256, 2, [(520, 600)], 0), (128, 4, [(2100, 2100), (3, 70)], 0),
    (64, 4, [(1100, 1111), (40, 40)], 130)])
def test_prompts_that_fill_the_chip(box, hd, group, lens, window):
    page, kv = 32, 8
    _say(f"attention e4m3 of prompts hd={hd} {lens} window={window}")
    rng = np.random.default_rng(35)
    b = paged.Batch(lens, page, rng, behind=1)
    pool = paged_more.Pool(kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
    heads = kv * group
    q = (1.5 * rng.standard_normal((b.n_tokens, heads, hd))).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(np.full_like(q, 7))
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, hd ** -0.5, window=window), box.dev.last_error()
    got = box.down(d_o, q)
    assert (got[-1] == 7).all() and np.isfinite(got).all()
    last = b.n_tokens - 2
    rows = sorted({0, 1, 15, 16, 31, 32, 63, 64, 500, 519, last} | set(rng.integers(0, last, 10).tolist()))
    want, bound = paged_more.attend(pool, _Some(b, rows), q, heads, hd ** -0.5, window)
    assert (np.abs(got[rows] - want[rows]).max((1, 2)) <= bound[rows]).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_missing_pages_and_nan(box, rows):
    """A page that is none poisons the rows that see it, a NaN of one sequence's stays there, a garbage scale byte of a
    block that nobody sees does nothing."""
    hd, page, kv, group = 64, 16, 1, 2
    _say(f"attention e4m3 missing pages rows={rows}")
    rng = np.random.default_rng(3)
    b = paged.Batch([(rows, 100), (rows, 100), (rows, 100)], page, rng)
    pool = paged_more.Pool(kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
    b.table[1, 1] = -1
    page_id, off = b.spot(2, 30)
    codes = pool.parts("k")[0]
    codes[page_id, :, off] = 127
    q = rng.standard_normal((b.n_tokens, kv * group, hd)).astype(np.float32)
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(q)
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, kv * group, 0.1), box.dev.last_error()
    got = box.down(d_o, q)
    assert np.isnan(got[rows:]).all()
    want, bound = paged_more.attend(pool, _Some(b, list(range(rows))), q, kv * group, np.float64(np.float32(0.1)))
    assert (np.abs(got[:rows] - want[:rows]).max((1, 2)) <= bound[:rows]).all()


@pytest.mark.parametrize("rows", [1, 200])
def test_pages_past_32_bits(box, rows):
    hd, page, kv, group = 256, 256, 8, 1
    _say(f"far pages e4m3 rows={rows}")
    rng = np.random.default_rng(33)
    heads, kind = kv * group, E4M3
    b = paged.Batch([(rows, rows + 100)], page, rng, spare=0)
    pool = paged_more.Pool(kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
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
    b.table = np.where(b.table >= 0, b.table - far, -1)
    qkv = rng.standard_normal((b.n_tokens, (heads + 2 * kv) * hd)).astype(np.float32)
    like = np.zeros((b.n_tokens, heads, hd), np.float32)
    d_q, d_o = box.up(like), box.up(like)
    assert box.dev.paged_append_enqueue(cache, batch, box.up(qkv), d_q, heads, EPS, BASE), box.dev.last_error()
    assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, hd ** -0.5), box.dev.last_error()
    paged_more.append(pool, b, qkv, heads, EPS, BASE)
    got = np.empty_like(pool.k), np.empty_like(pool.v)
    box.dev.dev_download(got[0], k + far * page_bytes)
    box.dev.dev_download(got[1], v + far * page_bytes)
    _same(got, pool, hd, page)
    q, out = box.down(d_q, like), box.down(d_o, like)
    few = sorted({0, rows // 2, rows - 1})
    want, bound = paged_more.attend(pool, _Some(b, few), q, heads, hd ** -0.5)
    assert (np.abs(out[few] - want[few]).max((1, 2)) <= bound[few]).all()


def test_captured_steps(box):
    """Append and attention in a graph, replayed as the sequences grow through their blocks, each replay against the
    eager calls over a copy of the cache."""
    hd, page, kv, group = 128, 16, 2, 4
    dev, heads, kind = box.dev, kv * group, E4M3
    _say("paged graph e4m3")
    rng = np.random.default_rng(12)
    b = paged.Batch([(1, 130), (1, 60), (1, 300)], page, rng)
    pool = paged_more.Pool(kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
    like = np.zeros((3, heads, hd), np.float32)
    batch = box.batch(b)
    caches = [box.cache(pool) for _ in range(2)]
    d_qkv, d_q, outs = box.up(np.zeros((3, (heads + 2 * kv) * hd), np.float32)), box.up(like), [box.up(like), box.up(like)]

    def step(i):
        assert dev.paged_append_enqueue(caches[i], batch, d_qkv, d_q, heads, EPS, BASE), dev.last_error()
        assert dev.paged_attention_enqueue(caches[i], batch, d_q, outs[i], heads, hd ** -0.5), dev.last_error()

    dev.dev_upload(box.kv_len, np.array([1, 1, 1], np.int32))
    step(0)
    step(1)
    assert dev.capture_begin(), dev.last_error()
    step(0)
    g = dev.capture_end()
    assert g, dev.last_error()
    try:
        for i in range(20):
            dev.dev_upload(box.kv_len, np.array([40 + i, 15 + i, 250 + i], np.int32))
            dev.dev_upload(d_qkv, (10.0 ** rng.uniform(-3, 2) * rng.standard_normal((3, (heads + 2 * kv) * hd))).astype(np.float32))
            dev.graph_launch(g, 1)
            step(1)
            np.testing.assert_array_equal(box.down(outs[0], like), box.down(outs[1], like))
            for side in "kv":
                x, y = (box.down(getattr(c.c, side), pool.k) for c in caches)
                np.testing.assert_array_equal(x, y)
    finally:
        dev.graph_destroy(g)
