"""A serving loop with adapters, drafts and endless streams, as a program would run it: the
projections with each request's adapter beside them, the append to an e4m3 cache, attention
by a window beside sinks (pages between given back), the head's product, and the
verification of the drafts; prompts, then steps of a few tokens a sequence, eager and from a
captured graph.  Each stage is held to its 64-bit definition over what the stage before gave."""
import numpy as np
import pytest

from tests import paged, paged_more
from tests.test_gpu_lora import Case as Lora
from tests.test_gpu_lora import check as check_lora
from tests.test_gpu_paged import _Box, _say
from tests.test_gpu_verify import Case as Verify
from zlm_amd import device as zd

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, HD, PAGE, VOCAB = 512, 8, 2, 64, 16, 4160
PACKED = (HEADS + 2 * KV) * HD
EPS, BASE, SCALE = 1e-6, 1e4, HD ** -0.5
ADAPTERS, RANK, DRAFTS = 3, 16, 3


@pytest.fixture
def box(dev):
    b = _Box(dev)
    yield b
    b.free()


class _Layer:
    """Weights, adapters, activations and the calls of one step over a batch."""

    def __init__(self, box, rng, n_max, n_seqs):
        self.box, self.dev = box, box.dev
        synth = lambda rows, seed: self.dev.synth_resident(zd.Q4_0, rows * HIDDEN // 32, seed, 0.02)  # noqa: E731
        self.w_qkv, self.w_o, self.w_lm = synth(PACKED, 1), synth(HIDDEN, 2), synth(VOCAB, 3)
        self.qn, self.kn = (1 + 0.1 * rng.standard_normal((2, HD))).astype(np.float32)
        self.d_qn, self.d_kn = box.up(self.qn), box.up(self.kn)
        # adapters of q alone (a part of the packed product's rows), and of the output
        self.lora_q = Lora(zd.BF16, n_max, ADAPTERS, RANK, HEADS * HD, HIDDEN, rng, ranks=[16, 5, 0], scales=[0.5, 2, 1])
        self.lora_o = Lora(zd.F16, n_max, ADAPTERS, RANK, HIDDEN, HEADS * HD, rng)
        self.q_pool, self.o_pool = self.lora_q.up(box), self.lora_o.up(box)
        zeros = lambda *s: box.up(np.zeros((n_max, *s), np.float32))  # noqa: E731
        self.x, self.base, self.qkv, self.q = zeros(HIDDEN), zeros(PACKED), zeros(PACKED), zeros(HEADS, HD)
        self.o, self.h0, self.h, self.logits = zeros(HEADS, HD), zeros(HIDDEN), zeros(HIDDEN), zeros(VOCAB)
        self.adapter = box.up(np.full(n_max, -1, np.int32))
        self.temp, self.u, self.u_draw = box.up(np.full(n_max, 0.8, np.float32)), zeros(), zeros()
        self.top_k = box.up(np.full(n_max, 40, np.int32))
        self.draft, self.token = box.up(np.zeros(n_max, np.int32)), box.up(np.full(n_max, -9, np.int32))
        self.accepted = box.up(np.full(n_seqs, -9, np.int32))

    def run(self, cache, batch, n, n_seqs, window, sinks, verify):
        d, mm = self.dev, zd.quant(zd.Q4_0)
        assert d.mat_mul_enqueue(self.w_qkv, mm, PACKED, HIDDEN, n, self.x, self.base), d.last_error()
        assert d.dev_copy_enqueue(self.qkv, self.base, 4 * n * PACKED), d.last_error()
        assert d.lora_enqueue(self.q_pool, n, self.adapter, self.x, self.qkv, res=self.qkv, y_stride=PACKED), d.last_error()
        assert d.paged_append_enqueue(cache, batch, self.qkv, self.q, HEADS, EPS, BASE, q_norm_w=self.d_qn,
                                      k_norm_w=self.d_kn), d.last_error()
        assert d.paged_attention_enqueue(cache, batch, self.q, self.o, HEADS, SCALE, window=window, sinks=sinks), d.last_error()
        assert d.mat_mul_enqueue(self.w_o, mm, HIDDEN, HEADS * HD, n, self.o, self.h0), d.last_error()
        assert d.lora_enqueue(self.o_pool, n, self.adapter, self.o, self.h, res=self.h0), d.last_error()
        if verify:
            assert d.mat_mul_enqueue(self.w_lm, mm, VOCAB, HIDDEN, n, self.h, self.logits), d.last_error()
            how = zd.Sampling(temperature=self.temp, top_k=self.top_k)
            assert d.verify_enqueue(self.logits, n, VOCAB, n_seqs, self.box.q_start, self.draft, self.u, self.u_draw,
                                    self.accepted, self.token, how=how), d.last_error()

    def free(self):
        self.dev.sync()
        for w in (self.w_qkv, self.w_o, self.w_lm):
            self.dev.free_resident(w)


def _lora_is(c, adapter, x, res, got):
    c.adapter, c.x, c.res = adapter, x, res
    check_lora(got, *c.want())


def _hold(box, layer, pool, b, adapter, window, sinks):
    n = int(b.q_start[-1])
    f32 = lambda p, *s: box.down(p, np.zeros((b.n_tokens, *s), np.float32))[:n]  # noqa: E731
    x, base, qkv = f32(layer.x, HIDDEN), f32(layer.base, PACKED), f32(layer.qkv, PACKED)
    _lora_is(layer.lora_q, adapter[:n], x, base[:, :HEADS * HD], qkv[:, :HEADS * HD])
    np.testing.assert_array_equal(qkv[:, HEADS * HD:], base[:, HEADS * HD:])
    q, o = f32(layer.q, HEADS, HD), f32(layer.o, HEADS, HD)
    want = paged_more.append(pool, b, box.down(layer.qkv, np.zeros((b.n_tokens, PACKED), np.float32)), HEADS, EPS, BASE,
                             layer.qn, layer.kn)[:n]
    np.testing.assert_allclose(q, want, rtol=2.0 ** -23, atol=1e-9)
    for side in "kv":
        np.testing.assert_array_equal(box.down(getattr(box, side), pool.k), getattr(pool, side))
    full = np.zeros((b.n_tokens, HEADS, HD), np.float32)
    full[:n] = q
    out, bound = paged_more.attend(pool, b, full, HEADS, SCALE, window, sinks)
    assert (np.abs(o - out[:n]).max((1, 2)) <= bound[:n]).all()
    h0, h = f32(layer.h0, HIDDEN), f32(layer.h, HIDDEN)
    _lora_is(layer.lora_o, adapter[:n], o.reshape(n, -1), h0, h)


def _hide(b, window, sinks):
    for s, (n, end) in enumerate(b.lens):
        first = max(0, end - n + 1 - window)
        lo, hi = -(-min(sinks, first) // b.page), first // b.page
        if hi > lo:
            b.table[s, lo:hi] = -1


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 5)])
def test_prompts_then_drafts(box, window, sinks):
    _say(f"more serving window={window} sinks={sinks}")
    rng = np.random.default_rng(31)
    dev, steps, n1 = box.dev, 5, 1 + DRAFTS
    prompts = [70, 9, 150, 33]
    seqs = len(prompts)
    room = paged.Batch([(1, n + n1 * steps) for n in prompts], PAGE, rng)
    b = paged.Batch([(n, n) for n in prompts], PAGE, rng, behind=2)
    b.table, b.stride, b.n_pages = room.table.copy(), room.stride, room.n_pages
    pool = paged_more.Pool(KV, HD, PAGE, room.n_pages, fill=rng)
    layer = _Layer(box, rng, b.n_tokens, seqs)
    request = np.array([0, -1, 2, 1], np.int32)
    cache, batch = box.cache(pool), box.batch(b)
    adapter = np.concatenate([np.repeat(request, prompts), [5, 5]]).astype(np.int32)
    dev.dev_upload(layer.adapter, adapter)
    dev.dev_upload(layer.x, rng.standard_normal((b.n_tokens, HIDDEN)).astype(np.float32))
    layer.run(cache, batch, b.n_tokens, seqs, window, sinks, verify=False)
    _hold(box, layer, pool, b, adapter, window, sinks)

    ends, graph = list(prompts), None
    step = paged.Batch([(n1, n + n1) for n in ends], PAGE, rng)
    step.table, step.stride, step.n_pages = room.table.copy(), room.stride, room.n_pages
    batch, n = box.batch(step), step.n_tokens
    adapter = np.repeat(request, n1).astype(np.int32)
    dev.dev_upload(layer.adapter, adapter)
    try:
        for i in range(steps):
            step.lens = [(n1, e + n1) for e in ends]
            step.kv_len = np.array([e for _, e in step.lens], np.int32)
            step.table = room.table.copy()
            if window:
                _hide(step, window, sinks)
            dev.dev_upload(box.kv_len, step.kv_len)
            dev.dev_upload(box.table, step.table)
            dev.dev_upload(layer.x, rng.standard_normal((n, HIDDEN)).astype(np.float32))
            u, u_draw = rng.random(n).astype(np.float32), rng.random(seqs).astype(np.float32)
            dev.dev_upload(layer.u, u)
            dev.dev_upload(layer.u_draw, u_draw)
            if graph is None:  # the first step is eager: layouts and scratch are made
                layer.run(cache, batch, n, seqs, window, sinks, verify=True)
                assert dev.capture_begin(), dev.last_error()
                layer.run(cache, batch, n, seqs, window, sinks, verify=True)
                graph = dev.capture_end()
                assert graph, dev.last_error()
                # drafts that the target likes: its own largest and a lesser one
            logits = box.down(layer.logits, np.zeros((n, VOCAB), np.float32))
            draft = np.argsort(-logits, 1)[np.arange(n), rng.integers(0, 3, n)].astype(np.int32)
            draft[1] = -1
            dev.dev_upload(layer.draft, draft)
            dev.graph_launch(graph, 2)  # twice: positions written again with the same values
            _hold(box, layer, pool, step, adapter, window, sinks)
            logits = box.down(layer.logits, np.zeros((n, VOCAB), np.float32))
            accepted = box.down(layer.accepted, np.zeros(seqs, np.int32))
            token = box.down(layer.token, np.zeros(n, np.int32))
            v = Verify([n1] * seqs, logits, draft, u, u_draw, how=dict(t=np.float32(0.8), k=40))
            assert v.rows == n
            v.check(accepted, token)
            # the eager step over the same state gives the same bits
            before = box.down(layer.h, np.zeros((n, HIDDEN), np.float32))
            layer.run(cache, batch, n, seqs, window, sinks, verify=True)
            np.testing.assert_array_equal(box.down(layer.h, before), before)
            np.testing.assert_array_equal(box.down(layer.token, token), token)
            np.testing.assert_array_equal(box.down(layer.accepted, accepted), accepted)
            # the accepted drafts stay; what lies behind them is written over by the next step
            ends = [e + 1 + int(a) for e, a in zip(ends, accepted)]
    finally:
        if graph:
            dev.graph_destroy(graph)
        layer.free()
