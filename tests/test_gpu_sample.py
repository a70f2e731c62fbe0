"""The sampler on the GPU against the definition in 64 bits: every filter alone and
together, sizes around the histogram's slices, equal logits, masked, infinite and
NaN ones, temperatures from 0 to infinity, and its use in a captured graph."""
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NAN, INF, MAX = np.nan, np.inf, np.finfo(np.float32).max


def _say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def draw(x, t, k, p, mp, u, shift=0.0):
    """(token, probability) of one row; shift: relative, of every threshold a weight is compared with."""
    x = x.astype(np.float64)
    ok = np.flatnonzero(x > -INF)
    if not len(ok):
        return -1, 0.0
    x = np.minimum(x, np.float64(MAX))
    order = ok[np.argsort(-x[ok], kind="stable")]
    if not t > 0:
        return int(order[0]), 1.0
    if k > 0:
        order = order[:k]
    t = min(np.float64(t), np.float64(MAX))
    w = np.exp((x[order] - x[order[0]]) / t)
    keep = np.ones(len(w), bool)
    if p < 1:
        before = np.cumsum(w) - w
        keep = before < np.float64(p) * (1 + shift) * w.sum()
        keep[0] = True
    if mp > 0:
        keep &= w >= min(np.float64(mp), 1.0)
    order, w = order[keep], w[keep]
    run = np.cumsum(w)
    at = min(int((run <= np.float64(u) * (1 + shift) * run[-1]).sum()), len(w) - 1)
    return int(order[at]), float(w[at] / run[-1])


class _Rows:
    def __init__(self, dev, logits, t=None, k=None, p=None, mp=None, u=None, stride=0):
        self.dev, self.bufs, self.n, self.vocab, self.stride = dev, [], logits.shape[0], logits.shape[1], stride
        if stride:
            wide = np.full((self.n, stride), 1e30, np.float32)
            wide[:, :self.vocab] = logits
            logits = wide
        up = lambda v, kind: 0 if v is None else self.up(np.broadcast_to(np.asarray(v, kind), self.n))  # noqa: E731
        self.logits = self.up(logits.astype(np.float32))
        self.t, self.k, self.p, self.mp = up(t, np.float32), up(k, np.int32), up(p, np.float32), up(mp, np.float32)
        self.u = up(u, np.float32)
        self.token, self.prob = self.up(np.full(self.n, -9, np.int32)), self.up(np.full(self.n, -9, np.float32))

    def up(self, a):
        a = np.ascontiguousarray(a)
        ptr = self.dev.dev_malloc(max(16, a.nbytes))
        self.bufs.append(ptr)
        self.dev.dev_upload(ptr, a)
        return ptr

    def enqueue(self):
        assert self.dev.sample_enqueue(self.logits, self.n, self.vocab, self.u, self.token, temperature=self.t,
                                       top_k=self.k, top_p=self.p, min_p=self.mp, prob=self.prob,
                                       stride=self.stride), self.dev.last_error()

    def results(self):
        token, prob = np.empty(self.n, np.int32), np.empty(self.n, np.float32)
        self.dev.dev_download(token, self.token)
        self.dev.dev_download(prob, self.prob)
        return token, prob

    def free(self):
        self.dev.sync()
        for ptr in self.bufs:
            self.dev.dev_free(ptr)


def _check(dev, logits, t=1.0, k=0, p=1.0, mp=0.0, u=0.5, exact=False, stride=0):
    """Tokens as the definition's.  A weight is held to 2^-35 of its bin's edge and what is e^-32 below the largest
    is left out: where a threshold lies that near a cumulative weight, the token on its other side is right too
    (not with `exact`: weights that are whole numbers)."""
    r = _Rows(dev, logits, t, k, p, mp, u, stride)
    r.enqueue()
    token, prob = r.results()
    r.free()
    n = logits.shape[0]
    args = [np.broadcast_to(np.asarray(v), n) for v in (t, k, p, mp, u)]
    for i in range(n):
        a = [v[i] for v in args]
        a = [np.float32(a[0]), int(a[1]), np.float32(a[2]), np.float32(a[3]), np.float32(a[4])]
        want, share = draw(logits[i].astype(np.float32), *a)
        eps = 2.0 ** -33 + logits.shape[1] * np.exp(-32)
        near = {want: share}
        if not exact:
            for s in (-eps, eps):
                tok, pr = draw(logits[i].astype(np.float32), *a, shift=s)
                near[tok] = pr
        assert int(token[i]) in near, (i, int(token[i]), near, a)
        # one rounding to f32 and the weights'
        assert abs(prob[i] - near[int(token[i])]) <= 2.0 ** -23 * abs(near[int(token[i])]) + 1e-30, (i, prob[i], near)
    return token


SIZES = [1, 2, 7, 63, 1000, 8191, 8192, 8193, 20000, 151936]


@pytest.mark.parametrize("vocab", SIZES)
@pytest.mark.parametrize("std", [0.3, 3.0, 30.0])
def test_filters(dev, vocab, std):
    _say(f"sample vocab={vocab} std={std}")
    rng = np.random.default_rng(vocab)
    rows = []
    for t in (0.6, 1.0, 1.7):
        for k in (0, 1, 2, 50, 3000, vocab, vocab + 5):
            for p, mp in ((1.0, 0.0), (0.9, 0.0), (0.3, 0.0), (1.0, 0.05), (0.95, 0.01), (0.999, 0.0)):
                rows.append((t, k, p, mp, rng.random()))
    rng.shuffle(rows)
    rows = np.array(rows[:24 if vocab > 10000 else 60])
    x = std * rng.standard_normal((len(rows), vocab))
    _check(dev, x, rows[:, 0], rows[:, 1].astype(np.int64), rows[:, 2], rows[:, 3], rows[:, 4].astype(np.float32),
           stride=0 if vocab % 2 else vocab + 3)


@pytest.mark.parametrize("vocab", [5, 1000, 8193, 40000])
def test_equal_logits_go_by_index(dev, vocab):
    """Whole-number weights: thresholds that meet a cumulative weight exactly are decided exactly."""
    _say(f"sample equal vocab={vocab}")
    u = np.array([0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.1, 0.9, 0.3], np.float32)
    for x in (0.0, -7.5, 1e-30, -MAX, 3e38):
        logits = np.full((8, vocab), x)
        _check(dev, logits, u=u, exact=True)
        _check(dev, logits, k=min(vocab, 4), u=u, exact=True)
        _check(dev, logits, p=0.5, u=u, exact=True)
        _check(dev, logits, mp=1.0, u=u, exact=True)
    # a bin of many logits of few values
    rng = np.random.default_rng(vocab)
    logits = 1.0 + rng.integers(0, 3, (8, vocab)) * 2.0 ** -20
    _check(dev, logits, p=0.7, u=u)
    _check(dev, logits, k=max(1, vocab // 2 + 1), u=u)
    _check(dev, logits, mp=0.9999999, u=u)


@pytest.mark.parametrize("std", [0.0005, 0.02])
def test_bins_of_many_tokens(dev, std):
    """More tokens of distinct values in a bin than are listed at once."""
    _say(f"sample crowded std={std}")
    rng = np.random.default_rng(4)
    x = 2.0 + std * rng.standard_normal((12, 60000))
    u = rng.random(12).astype(np.float32)
    _check(dev, x, u=u)
    _check(dev, x, k=rng.integers(1, 60000, 12), u=u)
    _check(dev, x, p=0.37, u=u)
    _check(dev, x, mp=float(np.exp(-2.5 * std)), u=u)
    _check(dev, np.round(x * 4096) / 4096, k=30001, p=0.9, mp=float(np.exp(-3 * std)), u=u)


def test_rounded_logits(dev):
    """Logits of 8 significant bits: many equal ones at every border."""
    rng = np.random.default_rng(6)
    x = (3 * rng.standard_normal((40, 33000))).astype(np.float32)
    x = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
    u = rng.random(40).astype(np.float32)
    _check(dev, x, t=0.8, k=rng.integers(1, 400, 40), u=u)
    _check(dev, x, t=1.3, p=rng.random(40).astype(np.float32), u=u)


def test_masked_and_special_logits(dev):
    _say("sample special")
    rng = np.random.default_rng(7)
    n, vocab = 12, 9000
    x = 3 * rng.standard_normal((n, vocab))
    x[0] = -INF                      # nothing to draw
    x[1] = NAN
    x[2, :] = -INF
    x[2, 8500] = -5                  # one token
    x[3, rng.random(vocab) < 0.9] = -INF
    x[4, rng.random(vocab) < 0.9] = NAN
    x[5, rng.random(vocab) < 0.9] = -MAX  # masked by the type's lowest value
    x[6] = -MAX                      # all of them
    x[7, 17] = INF
    x[8, [5, 8999]] = INF            # two that count alike
    x[9, :8192] = -INF               # a slice with nothing
    x[10] = np.where(np.arange(vocab) % 2, 0.0, -0.0)
    x[11] = -1e30 * np.abs(x[11])    # far below 0
    for u in (0.0, 0.3, 0.99):
        for t in (1.0, 0.0):
            token = _check(dev, x, t=t, u=u)
            assert token[0] == token[1] == -1 and token[2] == 8500
        _check(dev, x, t=0.7, k=5, p=0.9, mp=0.1, u=u)


def test_parameters_at_their_ends(dev):
    _say("sample parameter ends")
    rng = np.random.default_rng(8)
    x = 2 * rng.standard_normal((1, 12345)).repeat(10, 0)
    u = rng.random(10).astype(np.float32)
    for t in ([0.0, -1.0, NAN, 1e-45, 1e-30, 1e-3, 100.0, 1e30, INF, 0.5],):
        _check(dev, x, t=t, u=u)
    _check(dev, x, k=[0, -3, 1, 2, 12344, 12345, 12346, 2 ** 31 - 1, 4096, 4097], u=u)
    _check(dev, x, p=[0.0, -1.0, 1e-30, 0.5, 1.0, 2.0, NAN, 1 - 2.0 ** -24, 0.999, INF], u=u)
    _check(dev, x, mp=[0.0, -1.0, NAN, 1.0, 2.0, INF, 1e-45, 1e-10, 1 - 2.0 ** -24, 0.5], u=u)
    _check(dev, x, mp=0.3, t=[1e-45, 1e-30, 1e-3, 100.0, 1e30, INF, 0.5, 1.0, 2.0, 3.0], u=u)
    _check(dev, x, u=[0.0, 2.0 ** -24, 1 - 2.0 ** -24, 0.5, 0.25, 1e-20, 0.9, 0.99, 0.999, 0.9999])


def test_absent_parameters(dev):
    """No array leaves its filter off; the probability may be absent too."""
    rng = np.random.default_rng(9)
    x = (2 * rng.standard_normal((5, 4000))).astype(np.float32)
    u = rng.random(5).astype(np.float32)
    full = _check(dev, x, u=u)
    r = _Rows(dev, x, u=u)
    r.prob, prob = 0, r.prob
    r.enqueue()
    r.prob = prob
    token, prob = r.results()
    r.free()
    np.testing.assert_array_equal(token, full)
    assert (prob == -9).all()


def test_many_rows(dev):
    """More rows than one launch's histograms hold."""
    rng = np.random.default_rng(10)
    n, vocab = 900, 150000
    _say(f"sample rows={n}")
    base = (3 * rng.standard_normal(vocab)).astype(np.float32)
    logits = np.empty((n, vocab), np.float32)
    for i in range(n):
        logits[i] = np.roll(base, i)
    u = rng.random(n).astype(np.float32)
    r = _Rows(dev, logits, t=1.0, k=40, u=u)
    r.enqueue()
    token, _ = r.results()
    r.free()
    order = np.argsort(-base.astype(np.float64), kind="stable")[:40]
    run = np.cumsum(np.exp(base[order].astype(np.float64) - base[order[0]]))
    want = [(order[min(int((run <= np.float64(v) * run[-1]).sum()), 39)] + i) % vocab for i, v in enumerate(u)]
    np.testing.assert_array_equal(token, want)


def test_frequencies(dev):
    """Over a grid of uniform numbers every token comes as often as its probability says, to one count each way."""
    rng = np.random.default_rng(11)
    x = rng.standard_normal(50).astype(np.float32)
    n = 20000
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    r = _Rows(dev, np.broadcast_to(x, (n, 50)), t=0.9, u=u)
    r.enqueue()
    token, _ = r.results()
    r.free()
    w = np.exp(x.astype(np.float64) / np.float64(np.float32(0.9)))
    assert np.abs(np.bincount(token, minlength=50) - n * w / w.sum()).max() <= 2


def test_captured_draws(dev):
    """Replays read the logits and the numbers of their time, with eager draws of another size between."""
    rng = np.random.default_rng(12)
    x = (3 * rng.standard_normal((6, 20000))).astype(np.float32)
    u = rng.random(6).astype(np.float32)
    r = _Rows(dev, x, t=0.8, k=100, p=0.9, mp=0.01, u=u)
    other = _Rows(dev, x[:2, :9000], t=1.0, u=u[:2])
    r.enqueue()
    first = r.results()[0]
    assert dev.capture_begin(), dev.last_error()
    r.enqueue()
    g = dev.capture_end()
    assert g, dev.last_error()
    try:
        for i in range(3):
            y = np.roll(x, 37 * i, axis=1)
            dev.dev_upload(r.logits, np.ascontiguousarray(y))
            dev.dev_upload(r.token, np.full(6, -9, np.int32))
            dev.graph_launch(g, 2)
            got = r.results()
            other.enqueue()
            r.enqueue()
            want = r.results()
            np.testing.assert_array_equal(got[0], want[0])
            np.testing.assert_array_equal(got[1], want[1])
            if i == 0:
                np.testing.assert_array_equal(got[0], first)
    finally:
        dev.graph_destroy(g)
        r.free()
        other.free()
