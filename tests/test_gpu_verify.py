"""Verification of drafted tokens on the GPU against its definition in 64 bits: filters,
sizes around the histogram's slices, ragged batches, certain and drawn drafts, rows that
nothing can be drawn from, captured graphs, and the distribution of what comes out."""
import numpy as np
import pytest

from tests.test_gpu_paged import _Box, _say
from zlm_amd import device as zd

pytestmark = pytest.mark.gpu

INF = np.inf
MAX = np.float64(np.finfo(np.float32).max)


def shares(x, t=1.0, k=0, p=1.0, mp=0.0, shift=0.0):
    """The probability of every token of a row (float64; all 0 where there is none)."""
    x = x.astype(np.float64)
    out = np.zeros(len(x))
    ok = np.flatnonzero(x > -INF)
    if not len(ok):
        return out
    x = np.minimum(x, MAX)
    order = ok[np.argsort(-x[ok], kind="stable")]
    if not t > 0:
        out[order[0]] = 1
        return out
    if k > 0:
        order = order[:k]
    w = np.exp((x[order] - x[order[0]]) / min(np.float64(t), MAX))
    keep = np.ones(len(w), bool)
    if p < 1:
        keep = np.cumsum(w) - w < np.float64(p) * (1 + shift) * w.sum()
        keep[0] = True
    if mp > 0:
        keep &= w >= min(np.float64(mp), 1.0)
    out[order[keep]] = w[keep] / w[keep].sum()
    return out


class Case:
    """lens: rows of each sequence; how and draft_how: dicts of t, k, p, mp, each one value or one a row."""

    def __init__(self, lens, target, tokens, u, u_draw, draft=None, how=None, draft_how=None, behind=0):
        self.lens, self.target, self.draft = lens, target.astype(np.float32), draft
        self.q_start = np.cumsum([0] + list(lens)).astype(np.int32)
        self.rows, self.vocab = target.shape
        assert self.rows == self.q_start[-1] + behind
        self.tokens = np.asarray(tokens, np.int32)
        self.u, self.u_draw = np.asarray(u, np.float32), np.asarray(u_draw, np.float32)
        full = lambda how: {n: np.broadcast_to(np.asarray(v, np.int32 if n == "k" else np.float32), self.rows)  # noqa: E731
                            for n, v in (how or {}).items()}
        self.how, self.draft_how = full(how), full(draft_how)

    def _row(self, x, how, r, shift):
        a = {n: v[r] for n, v in how.items()}
        return shares(x[r], shift=shift, **a)

    def want(self, s, shift=0.0):
        """(accepted, the sequence's tokens); shift: relative, of every threshold."""
        r0, n = self.q_start[s], self.lens[s]
        got = []
        for i in range(n):
            p = self._row(self.target, self.how, r0 + i, shift)
            if i < n - 1:
                d = int(self.tokens[r0 + i])
                is_one = 0 <= d < self.vocab
                if is_one:
                    if self.draft is None:
                        q = np.zeros(self.vocab)
                        q[d] = 1
                    else:
                        q = self._row(self.draft.astype(np.float32), self.draft_how, r0 + i, shift)
                    if np.float64(self.u[r0 + i]) * q[d] < p[d] * (1 + shift):
                        got.append(d)
                        continue
                    rest = np.maximum(p - q, 0)
                    # (differences of shares that are equal but for their weights' rounding)
                    p = rest if (rest > 1e-9).any() or shift == 0 and rest.any() else p
            run = np.cumsum(p)
            live = np.flatnonzero(p > 0)
            at = -1
            if len(live):
                past = live[run[live] > np.float64(self.u_draw[s]) * run[-1] * (1 + shift)]
                at = int(past[0]) if len(past) else int(live[-1])
            return i, got + [at] + [-1] * (n - 1 - i)
        return 0, []

    def run(self, box, stride=0, draft_stride=0):
        def wide(x, by):
            if not by:
                return box.up(x.astype(np.float32))
            w = np.full((len(x), by), 1e30, np.float32)
            w[:, :x.shape[1]] = x
            return box.up(w)

        names = {"t": "temperature", "k": "top_k", "p": "top_p", "mp": "min_p"}
        sampling = lambda how: zd.Sampling(**{names[n]: box.up(v) for n, v in how.items()}) if how else None  # noqa: E731
        self.d_accepted = box.up(np.full(len(self.lens), -7, np.int32))
        self.d_token = box.up(np.full(self.rows, -9, np.int32))
        args = [wide(self.target, stride), self.rows, self.vocab, len(self.lens), box.up(self.q_start), box.up(self.tokens),
                box.up(self.u), box.up(self.u_draw), self.d_accepted, self.d_token]
        more = dict(how=sampling(self.how), draft_logits=0 if self.draft is None else wide(self.draft, draft_stride),
                    draft_how=sampling(self.draft_how), stride=stride, draft_stride=draft_stride)
        self.call = lambda: box.dev.verify_enqueue(*args, **more)
        assert self.call(), box.dev.last_error()
        return self.results(box)

    def results(self, box):
        return box.down(self.d_accepted, np.zeros(len(self.lens), np.int32)), box.down(self.d_token, np.zeros(self.rows, np.int32))

    def check(self, accepted, token, exact=False):
        """A weight is held to 2^-35 of its bin's edge, what is e^-32 below the largest left out: where a threshold lies
        that near, what the other side of it gives is right too."""
        eps = 2.0 ** -32 + 2 * self.vocab * np.exp(-32)
        for s, n in enumerate(self.lens):
            mine = int(accepted[s]), [int(t) for t in token[self.q_start[s]:self.q_start[s + 1]]]
            if mine == self.want(s):
                continue
            assert not exact, (s, mine, self.want(s))
            assert mine in [self.want(s, x) for x in (-eps, eps)], (s, n, mine, self.want(s))
        assert (token[self.q_start[-1]:] == -9).all()


def make(rng, lens, vocab, near=0.7, std=2.5, by_logits=True, how=None, draft_how=None, behind=0):
    rows = sum(lens) + behind
    x = (std * rng.standard_normal((rows, vocab))).astype(np.float32)
    y = (near * x + np.sqrt(1 - near ** 2) * std * rng.standard_normal((rows, vocab))).astype(np.float32)
    c = Case(lens, x, np.zeros(rows), rng.random(rows), rng.random(len(lens)), y if by_logits else None, how, draft_how,
             behind)
    if by_logits:
        for r in range(rows):
            q = c._row(y, c.draft_how, r, 0.0)
            c.tokens[r] = min(np.searchsorted(np.cumsum(q), rng.random() * q.sum(), side="right"), vocab - 1)
    else:
        c.tokens[:] = y.argmax(1)
    return c


@pytest.fixture
def box(dev):
    b = _Box(dev)
    yield b
    b.free()


LENS = [[1], [5], [3, 1, 0, 6, 2], [2] * 9]
HOWS = [None, dict(t=0.7), dict(t=1.3, k=50), dict(p=0.9), dict(k=20, p=0.8, mp=0.05), dict(mp=0.1), dict(t=0.0), dict(k=1)]


@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 1000, 8191, 8192, 8193, 20000])
@pytest.mark.parametrize("how", range(len(HOWS)))
@pytest.mark.parametrize("by_logits", [True, False])
def test_filters_and_sizes(box, vocab, how, by_logits):
    _say(f"verify vocab={vocab} how={HOWS[how]} by_logits={by_logits}")
    for i, lens in enumerate(LENS):
        rng = np.random.default_rng(vocab + 10 * how + i)
        c = make(rng, lens, vocab, near=(0.9, 0.5)[i % 2], std=(0.5, 3.0)[i // 2], by_logits=by_logits, how=HOWS[how],
                 draft_how=HOWS[(how + 3 * i) % len(HOWS)], behind=i)
        c.check(*c.run(box))


@pytest.mark.parametrize("vocab", [128256, 151936, 1 << 20])
@pytest.mark.parametrize("how", [0, 2, 3, 4])
def test_large_vocabularies(box, vocab, how):
    _say(f"verify vocab={vocab} how={HOWS[how]}")
    rng = np.random.default_rng(vocab % 1000 + how)
    for by_logits in (True, False):
        c = make(rng, [3, 2], vocab, near=0.95, by_logits=by_logits, how=HOWS[how], draft_how=HOWS[how])
        c.check(*c.run(box))


def test_each_row_its_own_filters(box):
    rng = np.random.default_rng(3)
    lens, vocab = [4, 4, 1, 7], 3000
    rows = sum(lens)
    pick = lambda *v: rng.choice(v, rows)  # noqa: E731
    how = dict(t=pick(0.0, 0.5, 1.0, 2.0), k=pick(0, 1, 30), p=pick(1.0, 0.7), mp=pick(0.0, 0.03))
    other = dict(t=pick(0.0, 0.9), k=pick(0, 5), p=pick(0.5, 0.99))
    c = make(rng, lens, vocab, how=how, draft_how=other)
    c.check(*c.run(box))


def test_strides(box):
    rng = np.random.default_rng(4)
    c = make(rng, [3, 2, 5], 1001, how=dict(k=40), draft_how=dict(p=0.9))
    c.check(*c.run(box, stride=1003, draft_stride=1101))
    got = c.run(box, stride=1001 * 7)
    c.check(*got)


def test_a_draft_like_the_target_is_accepted(box):
    rng = np.random.default_rng(5)
    for how in (dict(t=0.8, p=0.9), None, dict(k=10), dict(t=0.0)):
        c = make(rng, [6] * 20, 5000, near=1.0, how=how, draft_how=how)
        accepted, token = c.run(box)
        assert (accepted == 5).all()
        c.check(accepted, token)


def test_numbers_at_the_ends(box):
    """u of 0 accepts what has any weight, u just under 1 what has q's and more; draws at both ends of the order."""
    rng = np.random.default_rng(6)
    for u in (0.0, np.float32(1) - np.float32(2.0 ** -24)):
        for u_draw in (0.0, np.float32(1) - np.float32(2.0 ** -24)):
            for by_logits in (True, False):
                c = make(rng, [4, 1, 3], 700, by_logits=by_logits, how=dict(k=300))
                c.u[:], c.u_draw[:] = u, u_draw
                c.check(*c.run(box))


def test_what_is_no_draft_and_no_row(box):
    """Drafts outside the vocabulary, rows of -inf and NaN in target and draft, infinite logits, a draft of no weight."""
    rng = np.random.default_rng(7)
    vocab = 400
    for by_logits in (True, False):
        c = make(rng, [3] * 9 + [2], vocab, by_logits=by_logits, how=dict(p=0.95), draft_how=dict(p=0.95))
        for s, d in enumerate((-1, vocab, -2 ** 31, 2 ** 31 - 1)):
            c.tokens[3 * s + s % 2] = d
        c.target[12], c.target[15 + 1] = -INF, np.nan
        c.target[18, 5] = INF
        c.target[21] = np.where(rng.random(vocab) < 0.5, -INF, c.target[21])
        if by_logits:
            c.draft = c.draft.copy()
            c.draft[24] = -INF
            c.draft[25, c.tokens[25]] = -INF
        accepted, token = c.run(box)
        c.check(accepted, token)
        assert accepted[4] == 0 and token[12] == -1
        assert (accepted[:4] <= [0, 1, 0, 1]).all()


def test_equal_weights(box):
    """Logits of one value: shares that are whole parts, an acceptance that falls on its end."""
    vocab = 64
    target = np.zeros((4, vocab), np.float32)
    draft = np.where(np.arange(vocab) < 32, 0.0, -INF).astype(np.float32)[None].repeat(4, 0)
    c = Case([2, 2], target, [3, 0, 40, 0], [0.5, 0, 0.25, 0], [0.49, 0.26], draft)
    # p = 1/64, q = 1/32: 0.5 q is not under p; the rest lies on 32 .. 63.  40 has no q: accepted
    accepted, token = c.run(box)
    assert list(accepted) == [0, 1] and list(token) == [47, -1, 40, 16]
    # p = q but for a draft that is not accepted: u q < p holds for every u, so by a draft that is no token
    c = Case([2], target[:2], [-1, 0], [0.9, 0], [0.51], target[:2])
    accepted, token = c.run(box)
    assert list(accepted) == [0] and list(token) == [32, -1]


@pytest.mark.parametrize("how", [dict(k=7000), dict(p=0.3), dict(k=9000, p=0.5, mp=0.99), dict(mp=1.0)])
def test_cuts_among_more_tokens_than_are_listed(box, how):
    """Thousands of equal logits, or of nearly equal ones: more tokens in question than a workgroup lists."""
    rng = np.random.default_rng(8)
    for vocab in (12000, 30000):
        for by_logits in (True, False):
            c = make(rng, [3, 2], vocab, std=1e-3, near=0.5, by_logits=by_logits, how=how, draft_how=how)
            c.target[0], c.target[3] = 1.5, 0.0
            c.check(*c.run(box))


@pytest.mark.parametrize("n", [64, 65, 130, 300])
def test_many_drafts(box, n):
    rng = np.random.default_rng(n)
    c = make(rng, [n, 3], 50, near=0.999, std=1.0)
    c.u[:n - 2] = 0.0
    c.check(*c.run(box))


def test_many_sequences(box):
    rng = np.random.default_rng(11)
    lens = [1 + i % 4 if i % 97 else 0 for i in range(1024)]
    c = make(rng, lens, 300, how=dict(k=100), behind=3)
    c.check(*c.run(box))


def test_rows_go_in_rounds(box):
    """More rows and slices than the scratch holds histograms of: 180 rows of 32 slices of 6168 bytes, twice."""
    rng = np.random.default_rng(12)
    c = make(rng, [60] * 3, 1 << 18, near=0.99, how=dict(k=30), draft_how=dict(k=30))
    c.u[:] *= 0.3
    box.dev.launch_log(True)
    got = c.run(box)
    assert sum(r["what"] == "verify cuts" for r in box.dev.launch_log_read()) > 1
    box.dev.launch_log(False)
    c.check(*got)


def test_what_comes_out_has_the_targets_distribution(box):
    """The first token of 40 times 1024 sequences with one target and one draft: counts within five deviations of the
    target's shares (one in 10^6 of 20 tokens leaves them by chance; the numbers are the seed's)."""
    rng = np.random.default_rng(13)
    vocab, n, rounds = 20, 1024, 40
    x, y = rng.standard_normal((2, vocab)).astype(np.float32) * np.float32(1.5)
    q, p = shares(y), shares(x, t=0.8, k=15)
    counts = np.zeros(vocab)
    target, draft = np.repeat(x[None], 2 * n, 0), np.repeat(y[None], 2 * n, 0)
    for _ in range(rounds):
        tokens = np.zeros(2 * n, np.int32)
        tokens[::2] = np.searchsorted(np.cumsum(q), rng.random(n) * q.sum(), side="right")
        c = Case([2] * n, target, tokens, rng.random(2 * n), rng.random(n), draft, how=dict(t=0.8, k=15))
        _, token = c.run(box)
        counts += np.bincount(token[::2], minlength=vocab)
    total = n * rounds
    dev = np.sqrt(total * p * (1 - p))
    assert (np.abs(counts - total * p) <= 5 * dev).all(), (counts, total * p)
    assert (counts[p == 0] == 0).all()


def test_captured(box):
    """Two graphs over one scratch, with the sampler run between them, against eager calls; drafts and logits change."""
    dev = box.dev
    rng = np.random.default_rng(14)
    cases = [make(rng, [4, 2], 9000, how=dict(k=50)), make(rng, [3, 1, 5], 500, by_logits=False)]
    eager = [c.run(box) for c in cases]
    graphs = []
    for c in cases:
        assert dev.capture_begin(), dev.last_error()
        assert c.call(), dev.last_error()
        graphs.append(dev.capture_end())
        assert graphs[-1], dev.last_error()
    x = rng.standard_normal((3, 5000)).astype(np.float32)
    d_x, d_u, d_t = box.up(x), box.up(np.array([0.1, 0.5, 0.9], np.float32)), box.up(np.zeros(3, np.int32))
    try:
        for _ in range(3):
            for c, g, want in zip(cases, graphs, eager):
                dev.dev_upload(c.d_accepted, np.full(len(c.lens), -7, np.int32))
                dev.dev_upload(c.d_token, np.full(c.rows, -9, np.int32))
                dev.graph_launch(g, 2)
                for a, b in zip(c.results(box), want):
                    np.testing.assert_array_equal(a, b)
                assert dev.sample_enqueue(d_x, 3, 5000, d_u, d_t), dev.last_error()
                assert c.call(), dev.last_error()
                for a, b in zip(c.results(box), want):
                    np.testing.assert_array_equal(a, b)
    finally:
        for g in graphs:
            dev.graph_destroy(g)
