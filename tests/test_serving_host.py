"""What the serving operators' entry points refuse, launch and allocate, without a
GPU: the host library over the stand-in runtime (tests/fake_hip.cpp), whose
kernels do nothing.  Addresses are not read here."""
import ctypes

import numpy as np
import pytest

from tests import paged
from zlm_amd import device as zd
from tests.test_host_routes import FREES, MALLOCS, _Box, fake  # noqa: F401


@pytest.fixture
def box(fake):  # noqa: F811
    b = _Box(fake, 1 << 16, 1 << 16)
    b.mod = fake
    yield b
    b.dev.deinit()


def _cache(mod, k=1 << 20, v=1 << 21, type=zd.Q4_0, kv=2, hd=128, page=64, pages=4):
    return mod.PagedCache(k, v, type, kv, hd, page, pages)


def _batch(mod, seqs=2, tokens=3, q_start=1 << 12, kv_len=1 << 13, table=1 << 14, stride=2):
    return mod.PagedBatch(seqs, tokens, q_start, kv_len, table, stride)


BAD_CACHES = [dict(type=zd.Q8_0), dict(type=zd.F32), dict(hd=96), dict(hd=0), dict(kv=0), dict(kv=2000), dict(page=8),
              dict(page=48), dict(page=512), dict(page=0), dict(k=0), dict(v=0), dict(k=(1 << 20) + 8), dict(pages=0),
              dict(pages=0x80000000)]
BAD_BATCHES = [dict(seqs=1025), dict(tokens=(1 << 24) + 1), dict(q_start=0), dict(kv_len=0), dict(table=0),
               dict(stride=0)]


def _calls(box, cache, batch):
    d, p = box.dev, 1 << 16
    return {"append": lambda: d.paged_append_enqueue(cache, batch, p, p, 8, 1e-6, 1e6),
            "read": lambda: d.paged_read_enqueue(cache, batch, p, p),
            "attention": lambda: d.paged_attention_enqueue(cache, batch, p, p, 8, 0.1)}


@pytest.mark.parametrize("op", ["append", "read", "attention"])
def test_bad_caches_and_batches_are_refused(box, op):
    for bad in BAD_CACHES:
        assert not _calls(box, _cache(box.mod, **bad), _batch(box.mod))[op](), bad
        assert box.dev.last_error()
    for bad in BAD_BATCHES:
        assert not _calls(box, _cache(box.mod), _batch(box.mod, **bad))[op](), bad
        assert box.dev.last_error()
    assert _calls(box, _cache(box.mod), _batch(box.mod))[op](), box.dev.last_error()


def test_other_arguments_are_refused(box):
    d, p, c, b = box.dev, 1 << 16, _cache(box.mod), _batch(box.mod)
    for heads in (0, 3, 16386):
        assert not d.paged_attention_enqueue(c, b, p, p, heads, 0.1), heads
    for q, out in ((0, p), (p, 0), (p + 4, p), (p, p + 8)):
        assert not d.paged_attention_enqueue(c, b, q, out, 8, 0.1), (q, out)
    assert not d.paged_attention_enqueue(c, b, p, p, 8, 0.1, window=1 << 31)
    # 2^24 tokens of 128 q heads over sequences of 2^24 positions: more work than a call counts
    big = _batch(box.mod, seqs=1000, tokens=1 << 24, stride=1 << 18)
    assert not d.paged_attention_enqueue(_cache(box.mod, kv=8), big, p, p, 128, 0.1)
    assert "too large" in d.last_error()
    assert not d.paged_append_enqueue(c, b, 0, p, 8, 1e-6, 1e6)
    assert not d.paged_append_enqueue(c, b, p, 0, 8, 1e-6, 1e6)
    assert not d.paged_append_enqueue(c, b, p, p, 0, 1e-6, 1e6)
    assert not d.paged_append_enqueue(c, b, p, p, 8, 1e-6, 0.0)
    assert not d.paged_append_enqueue(c, b, p, p, 8, 1e-6, float("nan"))
    assert not d.paged_append_enqueue(c, b, p, p, 8, 1e-6, float("inf"))
    assert not d.paged_append_enqueue(c, b, p, p, 8, 1e-6, 1e6, q_norm_w=p)  # weights of q alone
    assert not d.paged_append_enqueue(c, b, p, p, 8, 1e-6, 1e6, qkv_stride=12 * 128 - 1)
    assert d.paged_append_enqueue(c, b, p, p, 8, 1e-6, 1e6, qkv_stride=12 * 128)
    assert not d.paged_read_enqueue(c, b, 0, p) and not d.paged_read_enqueue(c, b, p, 0)
    raw = box.raw
    assert not raw.zlm_gpu_paged_read_enqueue(d._h, None, ctypes.byref(b.c), p, p)
    assert not raw.zlm_gpu_paged_read_enqueue(d._h, ctypes.byref(c.c), None, p, p)


@pytest.mark.parametrize("op", ["append", "read", "attention"])
def test_tokens_of_a_batch_are_below_2_24(box, op):
    cache = _cache(box.mod)
    assert _calls(box, cache, _batch(box.mod, tokens=(1 << 24) - 1))[op](), box.dev.last_error()
    assert not _calls(box, cache, _batch(box.mod, tokens=1 << 24))[op]()
    assert "tokens" in box.dev.last_error()


def test_more_attention_than_a_call_counts_is_refused(box):
    """2^11 tokens of 128 q heads over tables of 2^24 positions; half of these is taken."""
    d, p, cache = box.dev, 1 << 16, _cache(box.mod, kv=1)
    ask = lambda stride: d.paged_attention_enqueue(  # noqa: E731
        cache, _batch(box.mod, seqs=10, tokens=1 << 11, stride=stride), p, p, 128, 0.1)
    assert not ask(1 << 18) and "too large for one call" in d.last_error()
    assert ask(1 << 17), d.last_error()


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 3e38])
def test_scales_without_a_product_are_refused(box, scale):
    """Scores times a NaN or an infinity (3e38 times log2 e is one) are in no order."""
    d, p = box.dev, 1 << 16
    assert not d.paged_attention_enqueue(_cache(box.mod), _batch(box.mod), p, p, 8, scale)
    assert "scale" in d.last_error()
    assert d.paged_attention_enqueue(_cache(box.mod), _batch(box.mod), p, p, 8, 2e38), d.last_error()


def test_an_empty_batch_launches_nothing(box):
    box.dev.launch_log(True)
    for empty in (dict(seqs=0), dict(tokens=0)):
        b = _batch(box.mod, q_start=0, kv_len=0, table=0, **empty)
        for op, call in _calls(box, _cache(box.mod, k=0, v=0), b).items():
            assert call(), (op, box.dev.last_error())
    assert box.dev.launch_log_read() == []


def test_attention_scratch_is_sized_eagerly(box):
    """Under capture the attention runs in the scratch that an eager call made, and fails without one."""
    d, call = box.dev, _calls(box, _cache(box.mod), _batch(box.mod))["attention"]
    assert d.capture_begin()
    assert not call() and "before capture" in d.last_error()
    d.graph_destroy(d.capture_end())
    assert call(), d.last_error()
    mallocs = box.stat(MALLOCS)
    assert d.capture_begin()
    assert call(), d.last_error()
    g = d.capture_end()
    assert call() and box.stat(MALLOCS) == mallocs
    # the scratch has room for every shape: calls of another beside the graph need no other
    wide = _calls(box, _cache(box.mod, hd=256), _batch(box.mod, seqs=1, tokens=300))["attention"]
    assert wide() and d.sample_enqueue(1 << 16, 800, 150000, 1 << 16, 1 << 16) and box.stat(MALLOCS) == mallocs
    d.graph_destroy(g)


def test_sampling_refusals(box):
    d, p = box.dev, 1 << 16
    assert d.sample_enqueue(p, 3, 1000, p, p, temperature=p, top_k=p, top_p=p, min_p=p, prob=p), d.last_error()
    assert d.sample_enqueue(p, 3, 1000, p, p, stride=1001), d.last_error()
    assert d.sample_enqueue(p, 3, 1 << 20, p, p), d.last_error()
    for vocab, more in ((0, {}), ((1 << 20) + 1, {}), (1000, dict(stride=999))):
        assert not d.sample_enqueue(p, 3, vocab, p, p, **more) and d.last_error()
    for bad in ((0, 3, 10, p, p), (p, 3, 10, 0, p), (p, 3, 10, p, 0)):
        assert not d.sample_enqueue(*bad) and "null" in d.last_error()
    d.launch_log(True)
    assert d.sample_enqueue(0, 0, 10, 0, 0) and d.launch_log_read() == []
    # rows in as many launches as the scratch takes
    assert d.sample_enqueue(p, 40000, 262144, p, p), d.last_error()
    launches = [r for r in d.launch_log_read() if r["what"] == "sample"]
    assert sum(r["grid_x"] for r in launches) == 40000 and len(launches) > 1
    assert d.scratch_device_bytes() <= 65 << 20
    raw = box.raw
    assert raw.zlm_gpu_sample_enqueue(d._h, p, 0, 1, 10, None, p, p, None)  # all filters off


def test_attention_workspace_is_made_eagerly(box):
    d, p = box.dev, 1 << 16
    call = _calls(box, _cache(box.mod), _batch(box.mod))["attention"]
    assert d.capture_begin()
    assert not call() and "before capture" in d.last_error()
    d.graph_destroy(d.capture_end())
    # the sampler's call makes the shared scratch, not the attention's counters
    assert d.sample_enqueue(p, 4, 1000, p, p)
    assert d.capture_begin()
    assert not call() and "eager call before capture" in d.last_error()
    d.graph_destroy(d.capture_end())
    assert call(), d.last_error()
    assert d.capture_begin()
    assert call(), d.last_error()
    d.graph_destroy(d.capture_end())


@pytest.mark.parametrize("first", ["attention", "sample"])
def test_serving_beside_a_captured_decode_step(box, first):
    """A graph of the contiguous caches' attention holds its scratch; the serving calls need none of it."""
    d, p = box.dev, 1 << 16
    calls = {"attention": _calls(box, _cache(box.mod), _batch(box.mod))["attention"],
             "sample": lambda: d.sample_enqueue(p, 4, 150000, p, p)}
    contiguous = lambda: d.attention_enqueue(p, p, p, 8, 2, 128, p, 64, 0.1, p)  # noqa: E731
    assert contiguous(), d.last_error()
    assert d.capture_begin() and contiguous()
    g = d.capture_end()
    assert g, d.last_error()
    held, freed = d.scratch_device_bytes(), box.stat(FREES)
    for name in sorted(calls, key=lambda n: n != first):
        assert calls[name](), (name, d.last_error())
    assert d.scratch_device_bytes() >= held + (64 << 20) and box.stat(FREES) == freed
    # nor do graphs of theirs hold the contiguous attention's
    d.graph_destroy(g)
    assert d.capture_begin() and all(call() for call in calls.values()), d.last_error()
    g = d.capture_end()
    assert d.attention_enqueue(p, p, p, 8, 2, 128, p, 4096, 0.1, p), d.last_error()
    d.graph_destroy(g)


def test_sampling_scratch_is_sized_eagerly(box):
    d, p = box.dev, 1 << 16
    assert d.capture_begin()
    assert not d.sample_enqueue(p, 4, 150000, p, p) and "sampling scratch" in d.last_error()
    d.graph_destroy(d.capture_end())
    assert d.sample_enqueue(p, 4, 150000, p, p)
    assert d.capture_begin()
    assert d.sample_enqueue(p, 4, 150000, p, p), d.last_error()
    d.graph_destroy(d.capture_end())


@pytest.mark.parametrize("type,seqs,tokens,group,want", [
    # one token a sequence, and few tokens each: the few-row kernel alone
    (zd.Q4_0, 1, 1, 4, ["few"]), (zd.Q4_0, 64, 64, 8, ["few"]), (zd.Q4_0, 8, 40, 4, ["few"]),
    (zd.Q4_0, 2, 2, 33, ["few"]), (zd.F16, 2, 2, 33, ["few"]), (zd.Q4_0, 1, 32, 4, ["few"]), (zd.F16, 1, 8, 4, ["few"]),
    # one sequence of more rows than it takes: the many-row kernel alone, its positions split while it has few items
    (zd.F16, 1, 9, 4, ["many", "merge"]), (zd.Q4_0, 1, 33, 4, ["many", "merge"]), (zd.Q4_0, 1, 2048, 4, ["many"]),
    (zd.Q4_0, 1, 300, 4, ["many", "merge"]),
    # prompts beside other sequences: both
    (zd.Q4_0, 16, 1015, 2, ["many", "merge", "few"]), (zd.F16, 200, 3000, 4, ["many", "few"]),
    (zd.Q4_0, 2, 4000, 4, ["many", "few"])])
def test_attention_routes(box, type, seqs, tokens, group, want):
    d, p = box.dev, 1 << 16
    d.launch_log(True)
    assert d.paged_attention_enqueue(_cache(box.mod, kv=8, type=type), _batch(box.mod, seqs=seqs, tokens=tokens), p, p,
                                     8 * group, 0.1), d.last_error()
    names = {"paged attention of many rows": "many", "paged attention of many rows, merge": "merge",
             "paged attention": "few"}
    log = d.launch_log_read()
    assert [names[r["what"]] for r in log if r["what"] in names] == want
    # a workgroup for every tile of 256 rows that the batch may make, kv head and split
    for r in log:
        if r["what"] == "paged attention of many rows":
            assert r["grid_x"] % 8 == 0 and r["grid_x"] // 8 >= -(-tokens * group // 256)


@pytest.mark.parametrize("type,seqs,tokens,group,want", [
    # drafts of a serving batch, and a short prompt in one: the few-row kernel alone
    (zd.Q4_0, 32, 160, 4, ["few"]), (zd.Q4_0, 64, 320, 4, ["few"]), (zd.F16, 32, 160, 4, ["few"]),
    (zd.F16, 64, 320, 4, ["few"]), (zd.Q4_0, 16, 215, 4, ["few"]), (zd.Q4_0, 64, 320, 8, ["few"]),
    # a longer prompt, also in a batch that has room for many sequences
    (zd.Q4_0, 64, 1363, 4, ["many", "few"]), (zd.Q4_0, 16, 465, 4, ["many", "merge", "few"]),
    (zd.Q4_0, 256, 2255, 4, ["many", "few"]), (zd.Q4_0, 1024, 2255, 4, ["many", "few"]),
    (zd.F16, 1024, 2255, 4, ["many", "few"])])
def test_attention_routes_of_drafts_and_prompts(box, type, seqs, tokens, group, want):
    test_attention_routes(box, type, seqs, tokens, group, want)


def test_page_bytes():
    assert zd.paged_page_bytes(zd.F16, 8, 128, 64) == 8 * 64 * 256
    assert zd.paged_page_bytes(zd.Q4_0, 8, 128, 64) == 8 * 64 * 72
    assert zd.paged_page_bytes(zd.Q4_0, 1, 64, 16) == 16 * 36
    for bad in ((zd.Q8_0, 8, 128, 64), (zd.F16, 8, 96, 64), (zd.F16, 8, 128, 24)):
        assert zd.paged_page_bytes(*bad) == 0


def test_page_bytes_of_heads_that_no_call_takes():
    assert zd.paged_page_bytes(zd.F16, 1024, 256, 256) == 1024 * 256 * 512
    for kv in (0, 1025, 2000, 0xFFFFFFFF):
        assert zd.paged_page_bytes(zd.F16, kv, 128, 64) == 0


def test_an_inert_device_refuses():
    dev = zd.Device()
    if dev.available():
        pytest.skip("a GPU is present")
    c, b = zd.PagedCache(16, 16, zd.F16, 1, 64, 16, 1), zd.PagedBatch(1, 1, 16, 16, 16, 1)
    assert not dev.paged_append_enqueue(c, b, 16, 16, 1, 1e-6, 1e6)
    assert not dev.paged_read_enqueue(c, b, 16, 16)
    assert not dev.paged_attention_enqueue(c, b, 16, 16, 1, 1.0)
    dev.deinit()


def test_rows_of_a_draw_up_to_32_bits(box):
    """The rows go in launches of some thousands: their count ends below 2^32 rows too."""
    d, p = box.dev, 1 << 16
    d.launch_log(True)
    assert d.sample_enqueue(p, (1 << 32) - 1, 1, p, p), d.last_error()
    rows = [r["grid_x"] for r in d.launch_log_read() if r["what"] == "sample"]
    assert len(set(rows[:-1])) == 1 and rows[0] > 1000
    d.launch_log(False)


@pytest.mark.parametrize("route", paged.TWO_PARTS)
def test_one_part_instead_of_two_shows(route):
    """The limit that the attention's routes are held to is under what one f16 part of q, or of the probabilities,
    would be off by: a mistake planted in the oracle."""
    x = paged.TwoParts(zd.F16, **paged.TWO_PARTS[route])
    want = x.want()
    for lost in (dict(q_parts=1), dict(p_parts=1)):
        assert np.nanmax(np.abs(x.want(**lost) - want)) > 4 * x.limit(), lost
    row = next(x.batch.places())
    x.batch.places = lambda: iter([row])
    full, _ = paged.attend(x.pool, x.batch, x.q, x.heads, np.float64(x.scale), x.window)
    assert np.abs(full[row[0]] - want[row[0]]).max() < 1e-12
