"""What the e4m3 cache and the attention with sinks refuse, launch and allocate, without a
GPU: the host library over the stand-in runtime (tests/fake_hip.cpp), whose kernels do
nothing.  Addresses are not read here."""
import pytest

from tests import paged, paged_more
from tests.test_host_routes import _Box, fake  # noqa: F401
from tests.test_serving_host import _batch, _cache
from zlm_amd import device as zd

E4M3 = zd.CACHE_E4M3


@pytest.fixture
def box(fake):  # noqa: F811
    b = _Box(fake, 1 << 16, 1 << 16)
    b.mod = fake
    yield b
    b.dev.deinit()


def test_bytes_of_a_page():
    for hd in (64, 128, 256):
        for page in (16, 32, 64, 128, 256):
            assert zd.paged_page_bytes(E4M3, 3, hd, page) == 3 * (page * hd + 16)
    assert zd.paged_page_bytes(E4M3, 3, 96, 16) == 0 and zd.paged_page_bytes(E4M3, 3, 64, 8) == 0
    assert zd.paged_page_bytes(E4M3, 1025, 64, 16) == 0 and zd.paged_page_bytes(E4M3 + 1, 1, 64, 16) == 0
    assert zd.paged_page_bytes(E4M3, 1024, 256, 256) == 1024 * (65536 + 16)


@pytest.mark.parametrize("bad", [dict(hd=96), dict(kv=0), dict(page=8), dict(page=48), dict(k=0), dict(v=0),
                                 dict(k=(1 << 20) + 8), dict(pages=0), dict(type=E4M3 + 1), dict(type=7)])
def test_bad_e4m3_caches_are_refused(box, bad):
    d, p, b = box.dev, 1 << 16, _batch(box.mod)
    cache = _cache(box.mod, **{"type": E4M3, **bad})
    assert not d.paged_append_enqueue(cache, b, p, p, 8, 1e-6, 1e6) and d.last_error()
    assert not d.paged_read_enqueue(cache, b, p, p) and d.last_error()
    assert not d.paged_attention_enqueue(cache, b, p, p, 8, 0.1) and d.last_error()
    assert not d.paged_attention_enqueue(cache, b, p, p, 8, 0.1, window=9, sinks=4) and d.last_error()
    good = _cache(box.mod, type=E4M3)
    assert d.paged_append_enqueue(good, b, p, p, 8, 1e-6, 1e6), d.last_error()
    assert d.paged_read_enqueue(good, b, p, p), d.last_error()
    assert d.paged_attention_enqueue(good, b, p, p, 8, 0.1), d.last_error()


@pytest.mark.parametrize("kind", [zd.F16, zd.Q4_0, E4M3])
def test_what_sinks_refuse(box, kind):
    d, p, b = box.dev, 1 << 16, _batch(box.mod)
    c = _cache(box.mod, type=kind)
    ask = lambda **how: d.paged_attention_enqueue(c, b, p, p, 8, 0.1, **how)  # noqa: E731
    assert ask(window=9, sinks=4), d.last_error()
    assert ask(sinks=4), d.last_error()
    assert ask(window=0x7fffffff, sinks=0x7fffffff), d.last_error()
    assert not ask(window=9, sinks=1 << 31) and "sinks" in d.last_error()
    assert not ask(window=1 << 31, sinks=4) and "window" in d.last_error()
    for q, out in ((0, p), (p, 0), (p + 4, p), (p, p + 8)):
        assert not d.paged_attention_enqueue(c, b, q, out, 8, 0.1, window=9, sinks=4), (q, out)
    assert not d.paged_attention_enqueue(c, b, p, p, 3, 0.1, window=9, sinks=4)
    assert not d.paged_attention_enqueue(c, b, p, p, 8, float("nan"), window=9, sinks=4)
    d.launch_log(True)
    for empty in (dict(seqs=0), dict(tokens=0)):
        e = _batch(box.mod, q_start=0, kv_len=0, table=0, **empty)
        assert d.paged_attention_enqueue(c, e, p, p, 8, 0.1, window=9, sinks=4), d.last_error()
        assert d.paged_append_enqueue(c, e, p, p, 8, 1e-6, 1e6), d.last_error()
    assert d.launch_log_read() == []


def test_sinks_take_the_scratch_that_the_attention_has(box):
    d, p, b, c = box.dev, 1 << 16, _batch(box.mod), _cache(box.mod, type=E4M3)
    assert d.capture_begin()
    assert not d.paged_attention_enqueue(c, b, p, p, 8, 0.1, window=9, sinks=4) and "before capture" in d.last_error()
    g = d.capture_end()
    if g:
        d.graph_destroy(g)
    assert d.paged_attention_enqueue(c, b, p, p, 8, 0.1), d.last_error()
    held = d.scratch_device_bytes()
    assert d.capture_begin()
    assert d.paged_attention_enqueue(c, b, p, p, 8, 0.1, window=9, sinks=4), d.last_error()
    g = d.capture_end()
    if g:
        d.graph_destroy(g)
    assert d.scratch_device_bytes() == held


def test_the_oracle_of_the_e4m3_cache():
    """The restatement itself: codes and numbers both ways, and a scale that holds its largest but no smaller one."""
    import numpy as np
    for byte in (paged_more.LEAST, 127, paged_more.MOST):
        codes = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
        x = paged_more.decode(codes, np.array(byte))
        np.testing.assert_array_equal(paged_more.encode(x, byte), codes)
        assert (x.astype(np.float16) == x).all()
    rng = np.random.default_rng(1)
    m = 10.0 ** rng.uniform(-6, 5, 1000)
    b = paged_more.scale_byte(m)
    assert ((m <= 448 * 2.0 ** (b - 127)) | (b == paged_more.MOST)).all()
    assert ((m > 448 * 2.0 ** (b - 128)) | (b == paged_more.LEAST)).all()
    near = paged_more.decode(paged_more.encode(m, b), b)
    held = (m <= 57344) & (m >= 2.0 ** (b.astype(float) - 127 - 6))
    assert (np.abs(near - m)[held] <= m[held] * 2.0 ** -4).all()
    assert list(paged_more.seen(9, 3, 2)) == [0, 1, 7, 8, 9] and list(paged_more.seen(3, 3, 9)) == [0, 1, 2, 3]
    assert paged.Pool(zd.F16, 1, 64, 16, 1).kind == zd.F16
