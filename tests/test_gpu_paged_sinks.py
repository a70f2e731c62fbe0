"""Attention over a paged cache by a window beside sinks, on the GPU against its 64-bit
restatement (tests/paged_more.py), for every cache type and on every route."""
import numpy as np
import pytest

from tests import paged, paged_more
from tests.test_gpu_paged import _Box, _say, _Some
from zlm_amd import device as zd

pytestmark = pytest.mark.gpu

TYPES = [zd.F16, zd.Q4_0, zd.CACHE_E4M3]


@pytest.fixture
def box(dev):
    b = _Box(dev)
    yield b
    b.free()


def _run(box, b, pool, q, heads, scale, window, sinks):
    cache, batch = box.cache(pool), box.batch(b)
    d_q, d_o = box.up(q), box.up(np.full_like(q, 7))
    ok = box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, scale, window=window, sinks=sinks)
    assert ok, box.dev.last_error()
    return box.down(d_o, q).astype(np.float64)


def _hide(b, window, sinks):
    """Takes away the pages that no row sees any position of."""
    for s, (n, end) in enumerate(b.lens):
        first = max(0, end - n + 1 - window)
        lo, hi = -(-min(sinks, first) // b.page), first // b.page
        if hi > lo:
            b.table[s, lo:hi] = -1


# rows and positions, window, sinks: none hidden; a gap of less than a block; sinks at the borders of blocks and pages;
# sinks that reach into the window; more sinks than positions; a row whose window hides all but sinks and itself
CASES = [
    ([(1, 1), (1, 5), (1, 40), (1, 300)], 8, 4),
    ([(1, 31), (1, 64), (1, 65), (1, 66), (1, 97), (1, 129), (1, 400)], 32, 32),
    ([(1, 200), (1, 333), (0, 9), (1, 1000)], 100, 70),
    ([(3, 150), (1, 151), (2, 90)], 50, 1000),
    ([(5, 500), (8, 8), (4, 2), (0, 0), (3, 0), (1, 700)], 1, 1),
    ([(37, 37), (20, 150), (5, 300), (1, 900)], 33, 5),
    ([(150, 400), (1, 3), (40, 700)], 90, 17),
    ([(130, 900)], 64, 64),
    ([(90, 90)], 16, 31),
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd,page,kv,group", [(128, 64, 2, 4), (64, 16, 3, 1), (256, 32, 1, 5), (128, 16, 1, 8),
                                              (128, 256, 1, 33)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_window_beside_sinks(box, kind, hd, page, kv, group, case):
    lens, window, sinks = CASES[case]
    _say(f"sinks kind={kind} hd={hd} page={page} kv={kv} group={group} case={case}")
    rng = np.random.default_rng(case * 23 + hd + group)
    heads = kv * group
    b = paged.Batch(lens, page, rng, behind=2)
    pool = paged_more.pool(kind, kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
    _hide(b, window, sinks)
    q = (1.5 * rng.standard_normal((b.n_tokens, heads, hd))).astype(np.float32)
    got = _run(box, b, pool, q, heads, hd ** -0.5, window, sinks)
    want, bound = paged_more.attend(pool, b, q, heads, hd ** -0.5, window, sinks)
    rows = ~np.isnan(want)
    assert (got[~rows] == 7.0).all()
    off = np.where(rows, np.abs(got - np.where(rows, want, 0)), 0).max((1, 2))
    assert (off <= bound).all(), (off.max(), bound[off.argmax()], int(off.argmax()))


# windows that the few-row kernel does not take alone: positions split over workgroups and joined
MANY = [([(150, 1700), (1, 3), (40, 1500)], 1100, 17), ([(140, 1400)], 1200, 64), ([(170, 1450), (3, 20)], 1064, 200),
        ([(130, 2000)], 1500, 1)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd,page,kv,group", [(128, 64, 1, 4), (64, 16, 2, 4), (256, 32, 1, 3)])
@pytest.mark.parametrize("case", range(len(MANY)))
def test_many_rows(box, kind, hd, page, kv, group, case):
    lens, window, sinks = MANY[case]
    _say(f"sinks many kind={kind} hd={hd} page={page} case={case}")
    rng = np.random.default_rng(case + hd)
    heads = kv * group
    b = paged.Batch(lens, page, rng, behind=1)
    pool = paged_more.pool(kind, kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
    _hide(b, window, sinks)
    q = (1.5 * rng.standard_normal((b.n_tokens, heads, hd))).astype(np.float32)
    assert box.dev.launch_log(True)
    got = _run(box, b, pool, q, heads, hd ** -0.5, window, sinks)
    assert "paged attention of many rows, merge" in [r["what"] for r in box.dev.launch_log_read()]
    box.dev.launch_log(False)
    assert (got[-1] == 7).all()
    last = b.n_tokens - 1
    rows = sorted({0, 1, 15, 16, 31, 32, 63, 64, 127, 128, lens[0][0] - 1, last - 1} & set(range(last)))
    want, bound = paged_more.attend(pool, _Some(b, rows), q, heads, hd ** -0.5, window, sinks)
    assert (np.abs(got[rows] - want[rows]).max((1, 2)) <= bound[rows]).all()
    assert np.isfinite(got).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd,group,lens,window,sinks", [
    (256, 2, [(1100, 2300), (1, 900)], 130, 40), (256, 2, [(520, 3000)], 700, 64), (128, 4, [(2100, 2400), (3, 700)], 300, 4),
    (64, 4, [(1100, 3000), (40, 400)], 129, 200)])
def test_prompts_that_fill_the_chip(box, kind, hd, group, lens, window, sinks):
    page, kv = 32, 8
    _say(f"sinks of prompts kind={kind} hd={hd} {lens}")
    rng = np.random.default_rng(35)
    b = paged.Batch(lens, page, rng, behind=1)
    pool = paged_more.pool(kind, kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
    _hide(b, window, sinks)
    heads = kv * group
    q = (1.5 * rng.standard_normal((b.n_tokens, heads, hd))).astype(np.float32)
    got = _run(box, b, pool, q, heads, hd ** -0.5, window, sinks)
    assert (got[-1] == 7).all() and np.isfinite(got).all()
    last = b.n_tokens - 2
    rows = sorted({0, 1, 15, 16, 31, 32, 63, 64, 500, 519, last} | set(rng.integers(0, last, 10).tolist()))
    want, bound = paged_more.attend(pool, _Some(b, rows), q, heads, hd ** -0.5, window, sinks)
    assert (np.abs(got[rows] - want[rows]).max((1, 2)) <= bound[rows]).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd,lens", [(128, [(1, 300), (2, 90), (1, 5000)]), (64, [(70, 700)]), (128, [(70, 700)]),
                                     (256, [(70, 700)]), (256, [(1, 500)])])
def test_more_window_than_positions_is_all(box, kind, hd, lens):
    """A window that hides nothing gives what no window does; sinks without a window change nothing."""
    page, kv, group = 32, 2, 4
    _say(f"sinks and all kind={kind} hd={hd} {lens}")
    rng = np.random.default_rng(1)
    b = paged.Batch(lens, page, rng)
    pool = paged_more.pool(kind, kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
    q = rng.standard_normal((b.n_tokens, kv * group, hd)).astype(np.float32)
    run = lambda w, s: _run(box, b, pool, q, kv * group, 0.1, w, s)  # noqa: E731
    want = run(0, 0)
    np.testing.assert_array_equal(run(0, 9), want)
    for w, s in ((1 << 20, 9), (0x7fffffff, 0x7fffffff), (40, 0x7fffffff)):
        np.testing.assert_array_equal(run(w, s), want)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_a_missing_sink_poisons(box, kind, rows):
    hd, page, kv, group = 64, 16, 1, 4
    _say(f"sinks missing kind={kind} rows={rows}")
    rng = np.random.default_rng(3)
    b = paged.Batch([(rows, 300), (rows, 300)], page, rng)
    pool = paged_more.pool(kind, kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
    _hide(b, 60, 20)
    b.table[1, 1] = b.n_pages  # positions 16 to 31: sinks among them
    q = rng.standard_normal((b.n_tokens, group, hd)).astype(np.float32)
    got = _run(box, b, pool, q, group, 0.1, 60, 20)
    assert np.isnan(got[rows:]).all()
    want, bound = paged_more.attend(pool, b, q, group, np.float64(np.float32(0.1)), 60, 20)
    assert (np.abs(got[:rows] - want[:rows]).max((1, 2)) <= bound[:rows]).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 40])
def test_last_positions(box, kind, hd, rows):
    """At the last position that a sequence can have (one page stands for all), and past it."""
    page, group, window, last = 256, 4, 40, (1 << 31) - 256
    _say(f"sinks at the last positions kind={kind} hd={hd} rows={rows}")
    rng = np.random.default_rng(hd + rows)
    b = paged.Batch([(rows, page)], page, rng, spare=0)
    pool = paged_more.pool(kind, 1, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
    q = rng.standard_normal((rows, group, hd)).astype(np.float32)
    stride = (1 << 31) // page
    kv_len, d_q, d_o = box.up(np.array([last], np.int32)), box.up(q), box.up(np.full_like(q, 7))
    batch = zd.PagedBatch(1, rows, box.up(np.array([0, rows], np.int32)), kv_len, box.up(np.zeros((1, stride), np.int32)),
                          stride)
    cache = box.cache(pool)

    def run():
        assert box.dev.paged_attention_enqueue(cache, batch, d_q, d_o, group, hd ** -0.5, window=window, sinks=70), \
            box.dev.last_error()
        return box.down(d_o, q)

    # the page's first 70 positions as sinks and its last ones as the window, as at 256 positions
    want, bound = paged_more.attend(pool, b, q, group, hd ** -0.5, window, 70)
    assert (np.abs(run() - want).max((1, 2)) <= bound).all()
    for past in (1, 255):
        box.dev.dev_upload(kv_len, np.array([last + past], np.int32))
        got = run()
        assert np.isnan(got[max(0, rows - past):]).all() and np.isfinite(got[:max(0, rows - past)]).all()


@pytest.mark.parametrize("kind", TYPES)
def test_captured_stream(box, kind):
    """A graph of one token a sequence, replayed as the streams go on and their windows leave pages behind."""
    hd, page, kv, group, window, sinks = 128, 16, 2, 4, 50, 5
    dev, heads = box.dev, kv * group
    _say(f"sinks graph kind={kind}")
    rng = np.random.default_rng(12)
    b = paged.Batch([(1, 400), (1, 300)], page, rng)
    pool = paged_more.pool(kind, kv, hd, page, b.n_pages)
    paged_more.fill(pool, b, rng)
    q = rng.standard_normal((2, heads, hd)).astype(np.float32)
    cache, batch, d_q, d_o = box.cache(pool), box.batch(b), box.up(q), box.up(q)
    whole = b.table.copy()

    def step():
        assert dev.paged_attention_enqueue(cache, batch, d_q, d_o, heads, 0.1, window=window, sinks=sinks), dev.last_error()

    step()
    assert dev.capture_begin(), dev.last_error()
    step()
    g = dev.capture_end()
    assert g, dev.last_error()
    try:
        for lens in ([3, 1], [56, 55], [57, 64], [200, 128], [399, 300]):
            b.lens, b.table = [(1, n) for n in lens], whole.copy()
            _hide(b, window, sinks)
            dev.dev_upload(box.kv_len, np.array(lens, np.int32))
            dev.dev_upload(box.table, b.table)
            want, bound = paged_more.attend(pool, b, q, heads, np.float64(np.float32(0.1)), window, sinks)
            got = []
            for run in (lambda: dev.graph_launch(g, 2), step, lambda: dev.graph_launch(g, 1)):
                dev.dev_upload(d_o, np.full_like(q, 9))
                run()
                got.append(box.down(d_o, q))
            for x in got:
                np.testing.assert_array_equal(x, got[0])
            assert (np.abs(got[0] - want).max((1, 2)) <= bound).all()
    finally:
        dev.graph_destroy(g)
