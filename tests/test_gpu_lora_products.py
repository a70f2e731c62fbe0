"""The products of adapters on the GPU, one at a time: A and B pick single numbers, so that a
result is one product of numbers with many bits, and each part of both has to take part.
Every rank's kernels, of few tokens and of many."""
import numpy as np
import pytest

from tests.test_gpu_lora import Case, TYPES, as_type, run
from tests.test_gpu_paged import _Box, _say
from zlm_amd import device as zd

pytestmark = pytest.mark.gpu

K = 320


@pytest.fixture
def box(dev):
    b = _Box(dev)
    yield b
    b.free()


class Picks:
    """Three adapters whose A and B have one number a row, in every place of the rank: row n of y is
    wb[n] wa[pick_r[n]] x[pick_k[pick_r[n]]]."""

    def __init__(self, kind, tokens, rank, rng):
        self.c = Case(kind, tokens, 3, rank, rank + 13, K, rng)
        self.c.res[:] = 0
        self.pick_k = rng.integers(0, K, (3, rank))
        self.pick_r = np.stack([rng.permutation(rank + 13) % rank for _ in range(3)])

    def set(self, x, wa, wb):
        c = self.c
        i, r, n = np.arange(3)[:, None], np.arange(c.rank)[None], np.arange(c.rows)[None]
        a, b = np.zeros((3, c.rank, K)), np.zeros((3, c.rows, c.rank))
        a[i, r, self.pick_k], b[i, n, self.pick_r] = wa, wb
        (c.a, c.a64), (c.b, c.b64) = as_type(a, c.kind), as_type(b, c.kind)
        assert (c.a64 == a).all() and (c.b64 == b).all()
        c.x = x.astype(np.float32)
        assert (c.x == x).all()
        w = c.adapter
        at = np.take_along_axis(self.pick_k, self.pick_r, 1)[w]
        wa, wb = np.broadcast_to(wa, (3, c.rank)), np.broadcast_to(wb, (3, c.rows))
        return np.take_along_axis(x, at, 1) * np.take_along_axis(wa, self.pick_r, 1)[w], wb[w]  # h of each row, and b


def odd(rng, bits, *shape):
    """Whole numbers of just so many bits."""
    return ((rng.integers(1 << (bits - 1), 1 << bits, shape) | 1) * rng.choice([-1, 1], shape)).astype(np.float64)


def dense(rng, *shape):
    """24 bits, half of the numbers with nearly all ones behind the first 8: what is cut off of a part is largest."""
    m = rng.integers(1 << 23, 1 << 24, shape)
    return (np.where(rng.random(shape) < 0.5, m | 0xFFF0, m) | 1) * rng.choice([-1.0, 1.0], shape)


RANKS = [40, 72, 136, 256]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rank", RANKS)
@pytest.mark.parametrize("tokens", [3, 100, 1100])
def test_exact_products(box, kind, rank, tokens):
    """24 bits of a number by weights of 1, and of a number and a weight together: exact in 32 bits, as is every sum of
    their parts' products."""
    _say(f"lora exact products kind={kind} rank={rank} tokens={tokens}")
    rng = np.random.default_rng(rank + tokens)
    p = Picks(kind, tokens, rank, rng)
    bits = {zd.F16: 11, zd.BF16: 8, zd.F32: 12}[kind]
    for x_bits, a_bits, b_bits in ((24, 1, 1), (24 - bits, bits, 1), (24 - bits, 1, bits)):
        x = np.ldexp(odd(rng, x_bits, tokens, K), rng.integers(-30, 30, (tokens, K)))
        h, b = p.set(x, odd(rng, a_bits, 3, rank), odd(rng, b_bits, 3, p.c.rows))
        want = h * b
        assert (want.astype(np.float32) == want).all() and want.all()
        np.testing.assert_array_equal(run(box, p.c), want)


@pytest.mark.parametrize("rank", [24] + RANKS)
@pytest.mark.parametrize("tokens", [3, 100, 300, 1100])
def test_products_of_24_bits(box, rank, tokens):
    """f32: a product of two numbers of 24 bits, in A x and in B h.  The parts of each are exact, and so are their
    products in 32 bits; that of both last parts is left out (each under 2^-15 of its number's first bit: 2^-30).  Seven
    additions, the smaller products first, are each off by less than a step (2^-23) of their sum, and sums before the
    last hold at most (2 2^-7 + 3 2^-14 + ..) of it: the two before the last count 2^-7 and 2 2^-7 of a step, those before
    less than 2^-10 together."""
    _say(f"lora 24 bits rank={rank} tokens={tokens}")
    rng = np.random.default_rng(rank * 7 + tokens)
    p = Picks(zd.F32, tokens, rank, rng)
    limit = 2.0 ** -23 * (1 + 3 * 2.0 ** -7 + 2.0 ** -10) + 2.0 ** -30
    for in_a in (True, False):
        x = np.ldexp(dense(rng, tokens, K), rng.integers(-30, 0, (tokens, K)))
        one = lambda n: rng.choice([-1.0, 1.0], (3, n))  # noqa: E731
        wide = lambda n: np.ldexp(dense(rng, 3, n), -23)  # noqa: E731
        h, b = p.set(x, wide(rank) if in_a else one(rank), one(p.c.rows) if in_a else wide(p.c.rows))
        want = h.astype(np.longdouble) * b.astype(np.longdouble)  # (h is rounded to 53 bits where in_a)
        off = np.abs((run(box, p.c) - want) / want)
        assert off.max() <= limit, (in_a, float(off.max() * 2.0 ** 23))


@pytest.mark.parametrize("tokens", [3, 1100])
def test_smallest_numbers(box, tokens):
    """Numbers down to the subnormal ones by weights of 1: a last part below 2^-133 is cut off, once in x and once in h."""
    _say(f"lora smallest tokens={tokens}")
    rng = np.random.default_rng(tokens)
    p = Picks(zd.F32, tokens, 24, rng)
    x = np.ldexp(dense(rng, tokens, K), -149 + rng.integers(0, 30, (tokens, K)))
    h, b = p.set(x, np.ones((3, 24)), np.ones((3, p.c.rows)))
    off = np.abs(run(box, p.c).astype(np.float64) - h)
    assert off.max() <= 2 * 2.0 ** -133
    assert off[np.abs(h) >= 2.0 ** -110].max() == 0
