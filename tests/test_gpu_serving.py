"""A layer of a serving loop as a program would run it: projection, append to the paged
cache, attention, projections, and the draw of the next tokens, for prompts and then for
steps of one token a sequence, eager and from a captured graph.  Each stage is held to
its 64-bit definition over what the stage before it gave."""
import numpy as np
import pytest

from tests import paged
from tests.test_gpu_paged import _Box, _say
from tests.test_gpu_sample import draw
from zlm_amd import device as zd

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, HD, PAGE, VOCAB = 512, 8, 2, 64, 16, 4160
PACKED = (HEADS + 2 * KV) * HD
EPS, BASE, SCALE = 1e-6, 1e4, HD ** -0.5


@pytest.fixture
def box(dev):
    b = _Box(dev)
    yield b
    b.free()


class _Layer:
    """Weights, activations and the calls of one step over a batch."""

    def __init__(self, box, kind, rng, n_max):
        self.box, self.dev = box, box.dev
        synth = lambda rows, seed: self.dev.synth_resident(zd.Q4_0, rows * HIDDEN // 32, seed, 0.02)  # noqa: E731
        self.w_qkv, self.w_o, self.w_lm = synth(PACKED, 1), synth(HIDDEN, 2), synth(VOCAB, 3)
        self.qn, self.kn = (1 + 0.1 * rng.standard_normal((2, HD))).astype(np.float32)
        self.d_qn, self.d_kn = box.up(self.qn), box.up(self.kn)
        zeros = lambda *s: box.up(np.zeros((n_max, *s), np.float32))  # noqa: E731
        self.x, self.qkv, self.q, self.o = zeros(HIDDEN), zeros(PACKED), zeros(HEADS, HD), zeros(HEADS, HD)
        self.h, self.logits = zeros(HIDDEN), zeros(VOCAB)
        self.u, self.temp, self.prob = zeros(), zeros(), zeros()
        self.top_p = box.up(np.full(n_max, 0.9, np.float32))
        self.top_k = box.up(np.full(n_max, 50, np.int32))
        self.token = box.up(np.full(n_max, -9, np.int32))

    def run(self, cache, batch, n, window, sample):
        d, mm = self.dev, zd.quant(zd.Q4_0)
        assert d.mat_mul_enqueue(self.w_qkv, mm, PACKED, HIDDEN, n, self.x, self.qkv), d.last_error()
        assert d.paged_append_enqueue(cache, batch, self.qkv, self.q, HEADS, EPS, BASE, q_norm_w=self.d_qn,
                                      k_norm_w=self.d_kn), d.last_error()
        assert d.paged_attention_enqueue(cache, batch, self.q, self.o, HEADS, SCALE, window=window), d.last_error()
        assert d.mat_mul_enqueue(self.w_o, mm, HIDDEN, HEADS * HD, n, self.o, self.h), d.last_error()
        if sample:
            assert d.mat_mul_enqueue(self.w_lm, mm, VOCAB, HIDDEN, n, self.h, self.logits), d.last_error()
            assert d.sample_enqueue(self.logits, n, VOCAB, self.u, self.token, temperature=self.temp, top_k=self.top_k,
                                    top_p=self.top_p, prob=self.prob), d.last_error()

    def free(self):
        self.dev.sync()
        for w in (self.w_qkv, self.w_o, self.w_lm):
            self.dev.free_resident(w)


def _hold(box, layer, pool, b, window):
    """q, the cache's new rows and the attention against the definitions over the device's qkv."""
    n = b.n_tokens
    qkv = box.down(layer.qkv, np.zeros((n, PACKED), np.float32))
    q = box.down(layer.q, np.zeros((n, HEADS, HD), np.float32))
    o = box.down(layer.o, np.zeros((n, HEADS, HD), np.float32))
    want = paged.append(pool, b, qkv, HEADS, EPS, BASE, layer.qn, layer.kn)
    live = ~np.isnan(want)
    np.testing.assert_allclose(q[live], want[live], rtol=2.0 ** -23, atol=1e-9)
    # the cache as it is now: the rows just written within a 4-bit step (an eighth of the block's largest) or an f16
    # one (2^-11) of the oracle's, whose own quotients may round the other way
    mine = {side: getattr(pool, side).copy() for side in "kv"}
    pool.k[...], pool.v[...] = box.down(box.k, pool.k), box.down(box.v, pool.v)
    for row, s, p in b.places():
        page, off = b.spot(s, p)
        got = pool.rows(np.array([page]), np.array([off]))
        theirs = {side: getattr(pool, side) for side in "kv"}
        pool.k, pool.v = mine["k"], mine["v"]
        ref = pool.rows(np.array([page]), np.array([off]))
        pool.k, pool.v = theirs["k"], theirs["v"]
        for x, y in zip(got, ref):
            step = np.abs(y) * 2.0 ** -10 + 2.0 ** -24
            if pool.kind == zd.Q4_0:
                step = np.abs(y).reshape(*y.shape[:-1], -1, 32).max(-1).repeat(32, -1) / 7
            assert (np.abs(x - y) <= step).all(), (row, s, p)
    out, bound = paged.attend(pool, b, q, HEADS, SCALE, window)
    off = np.where(live, np.abs(o - np.where(live, out, 0)), 0).max((1, 2))
    assert (off <= bound).all(), (off.max(), int(off.argmax()))
    return q, o


@pytest.mark.parametrize("kind", [zd.F16, zd.Q4_0])
@pytest.mark.parametrize("window", [0, 48])
def test_prompts_then_steps(box, kind, window):
    _say(f"serving kind={kind} window={window}")
    rng = np.random.default_rng(21)
    dev, steps = box.dev, 3
    prompts = [70, 9, 0, 150]
    # the table has room for the steps; a row of each kind behind the last sequence
    step = paged.Batch([(1 if n else 0, n + steps if n else 0) for n in prompts], PAGE, rng, behind=1)
    first = paged.Batch([(n, n) for n in prompts], PAGE, rng, behind=2)
    first.table, first.stride, first.n_pages = step.table, step.stride, step.n_pages
    pool = paged.Pool(kind, KV, HD, PAGE, step.n_pages)
    layer = _Layer(box, kind, rng, first.n_tokens)
    cache = box.cache(pool)
    batch = box.batch(first)
    dev.dev_upload(layer.x, rng.standard_normal((first.n_tokens, HIDDEN)).astype(np.float32))
    layer.run(cache, batch, first.n_tokens, window, sample=False)
    _hold(box, layer, pool, first, window)

    n = step.n_tokens
    batch = box.batch(step)  # q_start, kv_len and table of the steps
    temp = np.array([0.7, 0.0, 1.3, 1.0][:n], np.float32)
    dev.dev_upload(layer.temp, temp)
    graph = None
    try:
        for i in range(steps):
            lens = [(1, m + i + 1) if m else (0, 0) for m in prompts]
            step.lens = lens
            step.kv_len = np.array([e for _, e in lens], np.int32)
            dev.dev_upload(box.kv_len, step.kv_len)
            dev.dev_upload(layer.x, rng.standard_normal((n, HIDDEN)).astype(np.float32))
            u = rng.random(n).astype(np.float32)
            dev.dev_upload(layer.u, u)
            if graph is None:  # the first step is eager: layouts and scratch are made
                layer.run(cache, batch, n, window, sample=True)
                assert dev.capture_begin(), dev.last_error()
                layer.run(cache, batch, n, window, sample=True)
                graph = dev.capture_end()
                assert graph, dev.last_error()
            dev.dev_upload(layer.token, np.full(n, -9, np.int32))
            dev.graph_launch(graph, 2)  # twice: a position written again with the same values
            _, o = _hold(box, layer, pool, step, window)
            logits = box.down(layer.logits, np.zeros((n, VOCAB), np.float32))
            token = box.down(layer.token, np.zeros(n, np.int32))
            prob = box.down(layer.prob, np.zeros(n, np.float32))
            eps = 2.0 ** -33 + VOCAB * np.exp(-32)
            for r in range(n):
                near = [draw(logits[r], temp[r], 50, np.float32(0.9), 0.0, u[r], shift=s) for s in (0.0, -eps, eps)]
                assert int(token[r]) in [t for t, _ in near], (i, r)
                assert min(abs(prob[r] - p) for t, p in near if t == token[r]) <= 2.0 ** -23
            # the eager step over the same state gives the same bits
            layer.run(cache, batch, n, window, sample=True)
            np.testing.assert_array_equal(box.down(layer.o, o), o)
            np.testing.assert_array_equal(box.down(layer.token, token), token)
    finally:
        if graph:
            dev.graph_destroy(graph)
        layer.free()


def test_beside_a_captured_decode_step(dev):
    """A graph of the contiguous attention replays as before while the paged attention and the sampler, which had not
    run on this device object when it was captured, run eagerly between the replays."""
    own = zd.Device()
    assert own.available(), own.last_error()
    box = _Box(own)
    rng = np.random.default_rng(22)
    heads, kv, hd, seq = 8, 2, 128, 300
    q = rng.standard_normal((heads, hd)).astype(np.float32)
    k, v = rng.standard_normal((2, kv, seq, hd)).astype(np.float16)
    d_q, d_k, d_v, d_o = box.up(q), box.up(k), box.up(v), box.up(np.zeros_like(q))
    pos = box.up(np.array([seq - 1], np.int32))

    def contiguous():
        assert own.attention_enqueue(d_q, d_k, d_v, heads, kv, hd, pos, seq, hd ** -0.5, d_o), own.last_error()

    contiguous()
    first = box.down(d_o, q)
    assert np.isfinite(first).all() and first.any()
    assert own.capture_begin(), own.last_error()
    contiguous()
    g = own.capture_end()
    assert g, own.last_error()
    b = paged.Batch([(1, 200), (3, 40)], PAGE, rng)
    pool = paged.Pool(zd.F16, kv, hd, PAGE, b.n_pages)
    paged.fill(pool, b, rng)
    pq = rng.standard_normal((b.n_tokens, heads, hd)).astype(np.float32)
    cache, batch, d_pq, d_po = box.cache(pool), box.batch(b), box.up(pq), box.up(pq)
    x = rng.standard_normal((3, 5000)).astype(np.float32)
    u = np.array([0.1, 0.5, 0.9], np.float32)
    d_x, d_u, token = box.up(x), box.up(u), box.up(np.full(3, -9, np.int32))
    try:
        for _ in range(3):
            assert own.sample_enqueue(d_x, 3, 5000, d_u, token), own.last_error()
            assert own.paged_attention_enqueue(cache, batch, d_pq, d_po, heads, SCALE), own.last_error()
            own.dev_upload(d_o, np.zeros_like(q))
            own.graph_launch(g, 2)
            np.testing.assert_array_equal(box.down(d_o, q), first)
            want, bound = paged.attend(pool, b, pq, heads, SCALE)
            assert (np.abs(box.down(d_po, pq) - want).max((1, 2)) <= bound).all()
            got = box.down(token, np.zeros(3, np.int32))
            assert [int(t) for t in got] == [draw(x[r], 1.0, 0, 1.0, 0.0, u[r])[0] for r in range(3)]
    finally:
        own.graph_destroy(g)
        box.free()
        own.deinit()
