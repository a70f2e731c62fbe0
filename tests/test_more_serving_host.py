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


@pytest.mark.parametrize("kind", [zd.F16, zd.Q4_0, E4M3])
def test_which_kernels_take_sinks(box, kind):
    """The few-row kernel alone while its items are no more than its workgroups and windows short."""
    d, p, c = box.dev, 1 << 16, _cache(box.mod, type=kind, kv=8)

    def whats(tokens, seqs, **how):
        d.launch_log(True)
        assert d.paged_attention_enqueue(c, _batch(box.mod, seqs=seqs, tokens=tokens, stride=200), p, p, 32, 0.1, **how), \
            d.last_error()
        return [r["what"] for r in d.launch_log_read()]

    few, many = "paged attention", "paged attention of many rows"
    assert whats(256, 1, window=1000, sinks=100) == [few]
    assert whats(256, 4, window=64, sinks=4) == [few]
    assert many in whats(256, 1, window=1000, sinks=101)
    assert many in whats(257, 1, window=64, sinks=4)
    assert many in whats(256, 1, window=64)
    assert whats(4, 4, window=5000, sinks=4) == [few]


@pytest.mark.parametrize("kind", [zd.F16, zd.Q4_0, E4M3])
@pytest.mark.parametrize("hd,kv,heads,window,least,most", [
    (128, 1, 1, 64, 2048, 4096), (128, 1, 4, 64, 1024, 2048), (128, 1, 8, 1000, 512, 1024), (128, 8, 8, 1000, 512, 1024),
    (256, 1, 4, 64, 512, 1024), (256, 8, 8, 256, 512, 1024), (256, 8, 16, 64, 256, 512), (64, 8, 8, 64, 1024, 1025)])
def test_long_chunks_with_sinks(box, kind, hd, kv, heads, window, least, most):
    """An item of the few-row kernel walks from its sequence's window on, however short the window: chunks of `least`
    tokens are its, those of `most` and more the many-row kernel's."""
    d, p, c = box.dev, 1 << 16, _cache(box.mod, type=kind, kv=kv, hd=hd)
    for tokens in (64, 256, least, most, 2 * most, 8192):
        d.launch_log(True)
        assert d.paged_attention_enqueue(c, _batch(box.mod, seqs=1, tokens=tokens, stride=2000), p, p, heads, 0.1,
                                         window=window, sinks=4), d.last_error()
        many = "paged attention of many rows" in [r["what"] for r in d.launch_log_read()]
        assert many == (tokens >= most), tokens


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


LORA = dict(a=1 << 20, b=1 << 21, type=zd.BF16, n_adapters=5, rank=16, rows=100, k=64)


def _lora(mod, **how):
    return mod.Lora(**{**LORA, **how})


@pytest.mark.parametrize("bad", [dict(a=0), dict(b=0), dict(a=(1 << 20) + 8), dict(b=(1 << 21) + 2), dict(type=zd.Q4_0),
                                 dict(n_adapters=0), dict(n_adapters=4097), dict(rank=0), dict(rank=12), dict(rank=264),
                                 dict(rows=0), dict(rows=(1 << 24) + 1), dict(k=0), dict(k=48), dict(k=1 << 25)])
def test_bad_adapters_are_refused(box, bad):
    d, p = box.dev, 1 << 16
    assert not d.lora_enqueue(_lora(box.mod, **bad), 3, p, p, p + 4096, res=p + 8192), bad
    assert d.last_error()
    assert d.lora_enqueue(_lora(box.mod), 3, p, p, p + 4096, res=p + 8192), d.last_error()


def test_other_arguments_of_adapters(box):
    d, p, lora = box.dev, 1 << 16, _lora(box.mod)
    assert not d.lora_enqueue(lora, 3, 0, p, p) and not d.lora_enqueue(lora, 3, p, 0, p) and not d.lora_enqueue(lora, 3, p, p, 0)
    assert not d.lora_enqueue(lora, 3, p, p + 4, p)  # x by 16 bytes
    assert not d.lora_enqueue(lora, 3, p, p, p, x_stride=66)
    assert not d.lora_enqueue(lora, 3, p, p, p, x_stride=60) and not d.lora_enqueue(lora, 3, p, p, p, y_stride=99)
    assert d.lora_enqueue(lora, 3, p, p, p + 4, res=p + 4, x_stride=68, y_stride=101), d.last_error()
    d.launch_log(True)
    assert d.lora_enqueue(lora, 0, 0, 0, 0), d.last_error()
    assert d.launch_log_read() == []
    assert d.lora_enqueue(lora, 64, p, p, p), d.last_error()
    assert [r["what"] for r in d.launch_log_read()] == ["adapters down", "adapters up"]
    d.launch_log(True)
    assert d.lora_enqueue(lora, 256, p, p, p), d.last_error()
    assert [r["what"] for r in d.launch_log_read()] == ["adapters down", "adapters up"]
    d.launch_log(True)
    assert d.lora_enqueue(lora, 257, p, p, p), d.last_error()
    assert [r["what"] for r in d.launch_log_read()] == ["adapters, tokens grouped", "adapters down", "adapters up"]


@pytest.mark.parametrize("rank", [8, 256])
@pytest.mark.parametrize("n_adapters", [1, 4096])
@pytest.mark.parametrize("tokens", [1, 64, 65, 256, 512, 1024, 1025, 5000, 200000, 3000000])
def test_adapters_fit_the_scratch(box, rank, n_adapters, tokens):
    """Every launch's partials, tiles and order within the 64 MiB, whatever the sizes."""
    d, p = box.dev, 1 << 16
    lora = _lora(box.mod, n_adapters=n_adapters, rank=rank, k=4096)
    d.launch_log(True)
    assert d.lora_enqueue(lora, tokens, p, p, p + 16, res=p), d.last_error()
    done = 0
    for r in d.launch_log_read():
        if r["what"] != "adapters down":
            continue
        tiles, splits = r["grid_x"], r["grid_y"]
        assert tiles * splits * 16 * rank * 4 + 12 * tiles <= 64 << 20
        assert splits == 1 or tiles * splits <= 512
        done += 1
    assert done >= 1


def test_adapters_take_the_scratch_before_capture(box):
    d, p = box.dev, 1 << 16
    own = box.mod.Device()
    assert own.capture_begin()
    assert not own.lora_enqueue(_lora(box.mod), 3, p, p, p) and "before capture" in own.last_error()
    g = own.capture_end()
    if g:
        own.graph_destroy(g)
    assert own.lora_enqueue(_lora(box.mod), 3, p, p, p), own.last_error()
    held = own.scratch_device_bytes()
    assert own.sample_enqueue(p, 1, 100, p, p) and own.scratch_device_bytes() == held
    own.deinit()
    assert d.available()


def _verify(box, **how):
    p = 1 << 16
    a = dict(logits=p, rows=9, vocab=1000, n_seqs=2, q_start=p, draft=p, u=p, u_draw=p, accepted=p, token=p + 4096)
    a.update(how)
    return box.dev.verify_enqueue(a.pop("logits"), a.pop("rows"), a.pop("vocab"), a.pop("n_seqs"), a.pop("q_start"),
                                  a.pop("draft"), a.pop("u"), a.pop("u_draw"), a.pop("accepted"), a.pop("token"), **a)


@pytest.mark.parametrize("bad", [dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(stride=999), dict(draft_stride=999),
                                 dict(n_seqs=1025), dict(rows=65537), dict(logits=0), dict(q_start=0), dict(draft=0),
                                 dict(u=0), dict(u_draw=0), dict(accepted=0), dict(token=0), dict(token=1 << 16)])
def test_what_verification_refuses(box, bad):
    assert not _verify(box, **bad), bad
    assert box.dev.last_error()
    assert _verify(box), box.dev.last_error()
    assert _verify(box, draft_logits=1 << 20, how=box.mod.Sampling(top_k=1 << 16)), box.dev.last_error()


def test_launches_of_a_verification(box):
    d = box.dev
    d.launch_log(True)
    assert _verify(box, n_seqs=0, q_start=0, accepted=0), d.last_error()
    assert d.launch_log_read() == []
    assert _verify(box, rows=0, logits=0, draft=0, u=0, u_draw=0, token=0), d.last_error()
    assert [r["what"] for r in d.launch_log_read()] == ["verify draw"]
    d.launch_log(True)
    assert _verify(box), d.last_error()
    assert [(r["what"], r["grid_x"], r["grid_y"]) for r in d.launch_log_read()] == [
        ("verify histogram", 1, 9), ("verify cuts", 9, 1), ("verify draw", 1, 2)]
    d.launch_log(True)
    assert _verify(box, rows=65536, vocab=1 << 20, n_seqs=1024, draft_logits=1 << 16), d.last_error()
    log = d.launch_log_read()
    assert log[-1]["what"] == "verify draw" and (log[-1]["grid_x"], log[-1]["grid_y"]) == (256, 1024)
    kept = 2 * 65536 * 40 + 1024 * 256 * 16 + 1024 * 4
    for r in log:
        if r["what"] == "verify histogram":
            assert kept + r["grid_x"] * r["grid_y"] * (768 * 8 + 16) <= 64 << 20
    assert sum(r["grid_y"] for r in log if r["what"] == "verify histogram") == 2 * 65536


def test_verification_takes_the_scratch_before_capture(box):
    own = box.mod.Device()
    fresh = type("", (), {"dev": own})
    assert own.capture_begin()
    assert not _verify(fresh) and "before capture" in own.last_error()
    g = own.capture_end()
    if g:
        own.graph_destroy(g)
    assert _verify(fresh), own.last_error()
    own.deinit()
    assert box.dev.available()
