"""Low-rank adapters of many requests on the GPU against their definition in 64 bits: types,
ranks, sizes, strides, mixes of adapters, tokens without one, in place and not.  What a
pool holds behind an adapter's own rank is NaN."""
import numpy as np
import pytest

from tests.test_gpu_paged import _Box, _say
from zlm_amd import device as zd

pytestmark = pytest.mark.gpu

TYPES = [zd.F16, zd.BF16, zd.F32]


@pytest.fixture
def box(dev):
    b = _Box(dev)
    yield b
    b.free()


def bf16(x):
    """float32 to the nearest bf16, as its bits and as float64."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    h = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return h, (h.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def as_type(x, kind):
    """(what the device holds, its values in 64 bits)."""
    if kind == zd.BF16:
        return bf16(x)
    y = np.asarray(x, np.float16 if kind == zd.F16 else np.float32)
    return y, y.astype(np.float64)


class Case:
    """A pool, tokens and the definition's result."""

    def __init__(self, kind, tokens, n_adapters, rank, rows, k, rng, adapter=None, ranks=None, scales=None):
        self.kind, self.n, self.rank, self.rows, self.k = kind, n_adapters, rank, rows, k
        self.ranks = np.full(n_adapters, rank, np.int32) if ranks is None else np.asarray(ranks, np.int32)
        self.scales = None if scales is None else np.asarray(scales, np.float32)
        a = rng.standard_normal((n_adapters, rank, k)).astype(np.float32) * np.float32(k ** -0.5)
        b = rng.standard_normal((n_adapters, rows, rank)).astype(np.float32)
        for i, r in enumerate(self.ranks):
            a[i, max(r, 0):], b[i, :, max(r, 0):] = np.nan, np.nan
        with np.errstate(invalid="ignore"):
            (self.a, self.a64), (self.b, self.b64) = as_type(a, kind), as_type(b, kind)
        if kind == zd.BF16:  # the rounding above is for numbers
            self.a, self.b = np.where(np.isnan(a), np.uint16(0x7FC0), self.a), np.where(np.isnan(b), np.uint16(0x7FC0), self.b)
        self.x = rng.standard_normal((tokens, k)).astype(np.float32)
        self.res = rng.standard_normal((tokens, rows)).astype(np.float32)
        self.adapter = np.asarray(rng.integers(0, n_adapters, tokens) if adapter is None else adapter, np.int32)

    def want(self, res=True):
        """(y, a bound of the kernel's distance from it), float64.  A product of parts is exact or (f32) off by 2^-22 of
        it; every sum rounds once a product (three or six of parts each) and once for each of up to 8 waves and 16
        splits: 2^-24 of the sum of the sizes each."""
        y = self.res.astype(np.float64) if res else np.zeros(self.res.shape)
        bound = np.abs(y) * 2.0 ** -24
        parts = 3 if self.kind == zd.BF16 else 6
        for t, i in enumerate(self.adapter):
            if not 0 <= i < self.n or self.ranks[i] <= 0:
                continue
            r = min(self.ranks[i], self.rank)
            s = 1.0 if self.scales is None else np.float64(self.scales[i])
            x, a, b = self.x[t].astype(np.float64), self.a64[i, :r], self.b64[i, :, :r]
            h = a @ x
            e_h = (np.abs(a) @ np.abs(x)) * 2.0 ** -24 * (parts * self.k + 24 + 4)
            d = b @ h
            e_d = np.abs(b) @ (e_h + (np.abs(h) + e_h) * 2.0 ** -24 * (parts * r + 4))
            y[t] += s * d
            bound[t] += abs(s) * e_d + (np.abs(y[t]) + abs(s) * e_d) * 2.0 ** -23
        return y, bound

    def up(self, box):
        self.d_a, self.d_b = box.up(self.a), box.up(self.b)
        return zd.Lora(self.d_a, self.d_b, self.kind, self.n, self.rank, self.rows, self.k, ranks=box.up(self.ranks),
                       scales=0 if self.scales is None else box.up(self.scales))


def run(box, c, in_place=False, res=True):
    lora, d_ad, d_x, d_res = c.up(box), box.up(c.adapter), box.up(c.x), box.up(c.res)
    d_y = d_res if in_place else box.up(np.full_like(c.res, 7))
    assert box.dev.lora_enqueue(lora, len(c.x), d_ad, d_x, d_y, res=d_res if res else 0), box.dev.last_error()
    return box.down(d_y, c.res)


def check(got, want, bound):
    off = np.abs(got - want)
    assert (off <= bound).all(), (np.unravel_index(off.argmax(), off.shape), off.max(), (off / bound).max())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 128, 136, 256])
@pytest.mark.parametrize("tokens,n_adapters,rows,k", [(1, 3, 100, 64), (5, 2, 33, 32), (64, 5, 129, 288), (65, 70, 260, 96),
                                                      (300, 4, 515, 128), (1100, 4, 515, 64)])
def test_sizes(box, kind, rank, tokens, n_adapters, rows, k):
    _say(f"lora kind={kind} rank={rank} tokens={tokens} adapters={n_adapters} rows={rows} k={k}")
    rng = np.random.default_rng(rank + tokens)
    adapter = rng.integers(-2, n_adapters + 2, tokens)  # some have none
    ranks = rng.integers(0, rank + 1, n_adapters)
    ranks[0] = rank
    if tokens == 1:
        adapter[:] = 0
    c = Case(kind, tokens, n_adapters, rank, rows, k, rng, adapter, ranks, rng.uniform(-2, 2, n_adapters))
    want, bound = c.want()
    check(run(box, c), want, bound)
    check(run(box, c, in_place=True), want, bound)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tokens", [1, 16, 17, 63, 64, 65, 128, 1000, 1024, 1025, 1500])
@pytest.mark.parametrize("mix", ["one", "none", "each", "blocks", "two"])
def test_mixes(box, kind, tokens, mix):
    _say(f"lora kind={kind} tokens={tokens} mix={mix}")
    rng = np.random.default_rng(tokens)
    n = 40
    t = np.arange(tokens)
    adapter = {"one": t * 0 + 7, "none": t * 0 - 1, "each": t % n, "blocks": t // 19 % n, "two": np.where(t % 2, 3, -1)}[mix]
    c = Case(kind, tokens, n, 16, 68, 64, rng, adapter)
    want, bound = c.want()
    got = run(box, c)
    check(got, want, bound)
    if mix == "none":
        np.testing.assert_array_equal(got, c.res)
    check(run(box, c, in_place=True), want, bound)
    want, bound = c.want(res=False)
    check(run(box, c, res=False), want, bound)


@pytest.mark.parametrize("tokens", [65, 127, 192, 255, 256, 257])
@pytest.mark.parametrize("mix", ["one", "most", "ends", "thirds", "each"])
def test_tiles_at_the_borders(box, tokens, mix):
    """Tokens that a workgroup groups by itself, and one more: tiles that end with the tokens or with an adapter's, of
    pools as large as there are, adapters in any order."""
    _say(f"lora borders tokens={tokens} mix={mix}")
    rng = np.random.default_rng(tokens)
    n, rank, rows, k = 4096, 8, 20, 64
    t = np.arange(tokens)
    adapter = {"one": t * 0 + n - 1, "most": np.where(t % 32 == 31, t, 5), "ends": np.array([0, n - 1, n, -1])[t % 4],
               "thirds": np.where(t < 33, 2, np.where(t < 64, 1, 0)), "each": rng.permutation(n)[:tokens]}[mix]
    c = Case(zd.F16, tokens, n, rank, rows, k, rng, adapter, rng.integers(0, rank + 1, n), rng.uniform(-2, 2, n))
    want, bound = c.want()
    got = run(box, c)
    check(got, want, bound)
    np.testing.assert_array_equal(run(box, c), got)
    np.testing.assert_array_equal(run(box, c, in_place=True), got)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tokens", [3, 100, 1100])
def test_every_bit_of_a_number_counts(box, kind, tokens):
    """A and B pick single numbers: the result is exact where every part of x, of h and of the weights takes part (24
    bits of x by weights of 1; of the weights by x of 1 for f32; 13 bits by 11 for f16, 16 by 8 for bf16)."""
    k, rank, rows = 320, 24, 50
    _say(f"lora exact kind={kind} tokens={tokens}")
    rng = np.random.default_rng(3)
    c = Case(kind, tokens, 3, rank, rows, k, rng, scales=[1, 2, -0.5])
    pick_k, pick_r = rng.integers(0, k, (3, rank)), rng.integers(0, rank, (3, rows))
    i, r, n = np.arange(3)[:, None], np.arange(rank)[None], np.arange(rows)[None]
    odd = lambda bits, *shape: (rng.integers(1 << (bits - 1), 1 << bits, shape) | 1) * rng.choice([-1, 1], shape)  # noqa: E731
    for wide in range(3):  # the bits are in x, in A, in B
        bits = {zd.F16: 11, zd.BF16: 8, zd.F32: 24}[kind]
        wa, wb = odd(bits, 3, rank), odd(bits, 3, rows)
        x_bits = 24 if wide == 0 else 24 - bits
        x = odd(x_bits, tokens, k) if x_bits else rng.choice([-1, 1], (tokens, k))
        c.x = np.ldexp(x.astype(np.float64), rng.integers(-30, 30, (tokens, k))).astype(np.float32)
        a, b = np.zeros((3, rank, k)), np.zeros((3, rows, rank))
        a[i, r, pick_k] = wa if wide == 1 else 1
        b[i, n, pick_r] = wb if wide == 2 else 1
        (c.a, c.a64), (c.b, c.b64) = as_type(a, kind), as_type(b, kind)
        assert (c.a64 == a).all() and (c.b64 == b).all()
        c.res[:] = 0
        want, _ = c.want()
        assert (want.astype(np.float32) == want).all() and want.any()
        np.testing.assert_array_equal(run(box, c), want)


@pytest.mark.parametrize("tokens,rank,n_adapters,rows,k", [(1, 16, 2, 5000, 8192), (40, 64, 40, 1000, 4096), (3000, 128, 5, 300, 512),
                                                           (9000, 8, 3000, 40, 32)])
def test_larger(box, tokens, rank, n_adapters, rows, k):
    """k over several workgroups, many tiles, more adapters than tiles; some tokens are looked at."""
    _say(f"lora larger tokens={tokens} rank={rank} adapters={n_adapters} rows={rows} k={k}")
    rng = np.random.default_rng(tokens)
    c = Case(zd.BF16, tokens, n_adapters, rank, rows, k, rng)
    got = run(box, c)
    for t in sorted({0, tokens // 2, tokens - 1} | set(rng.integers(0, tokens, 30).tolist())):
        one = Case.__new__(Case)
        one.__dict__.update(c.__dict__, x=c.x[t:t + 1], res=c.res[t:t + 1], adapter=c.adapter[t:t + 1])
        want, bound = one.want()
        check(got[t:t + 1], want, bound)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tokens,rank", [(511, 256), (512, 256), (513, 256), (1023, 128), (1024, 128), (1025, 128)])
def test_between_few_and_many(box, kind, tokens, rank):
    """Where the tiles' size changes: adapters in any order, ranks of their own, rows of y that end within a span."""
    _say(f"lora few and many kind={kind} tokens={tokens} rank={rank}")
    rng = np.random.default_rng(tokens)
    n = 7
    c = Case(kind, tokens, n, rank, 150, 160, rng, rng.integers(-1, n, tokens), rng.integers(1, rank + 1, n))
    want, bound = c.want()
    check(run(box, c), want, bound)
    check(run(box, c, in_place=True), want, bound)


@pytest.mark.parametrize("kind", TYPES)
def test_rounds_of_the_scratch(box, kind):
    """More tokens and adapters of the largest rank than the scratch holds at once."""
    tokens, n, rank, rows, k = 6000, 4096, 256, 8, 32
    _say(f"lora rounds kind={kind}")
    rng = np.random.default_rng(4)
    c = Case(kind, tokens, n, rank, rows, k, rng, np.arange(tokens) * 7 % (n + 1))
    box.dev.launch_log(True)
    got = run(box, c)
    assert sum(r["what"] == "adapters down" for r in box.dev.launch_log_read()) > 1
    box.dev.launch_log(False)
    for t in rng.integers(0, tokens, 40):
        one = Case.__new__(Case)
        one.__dict__.update(c.__dict__, x=c.x[t:t + 1], res=c.res[t:t + 1], adapter=c.adapter[t:t + 1])
        check(got[t:t + 1], *one.want())


@pytest.mark.parametrize("rows,y_stride,at", [(100, 300, 8), (100, 301, 8), (99, 300, 8), (100, 300, 3), (64, 64, 0)])
@pytest.mark.parametrize("tokens", [9, 200, 300, 1100])
def test_parts_of_wider_rows(box, rows, y_stride, at, tokens):
    """y as some columns of a packed product's rows, x as some of wider ones; what lies beside them stays."""
    k, x_stride, rank = 64, 100, 16
    _say(f"lora strides rows={rows} stride={y_stride} at={at} tokens={tokens}")
    rng = np.random.default_rng(rows + at)
    c = Case(zd.F16, tokens, 3, rank, rows, k, rng, rng.integers(-1, 3, tokens))
    wide_x = rng.standard_normal((tokens, x_stride)).astype(np.float32)
    wide_x[:, 4:4 + k] = c.x
    wide = rng.standard_normal((tokens + 1, y_stride)).astype(np.float32)
    flat = wide.reshape(-1)
    cols = [flat[at + t * y_stride:at + t * y_stride + rows] for t in range(tokens)]
    c.res = np.stack(cols)
    want, bound = c.want()
    lora, d_ad, d_x = c.up(box), box.up(c.adapter), box.up(wide_x)
    d_res, d_y = box.up(wide), box.up(np.full_like(wide, 7))
    for res, y in ((d_res, d_y), (d_res, d_res)):
        assert box.dev.lora_enqueue(lora, tokens, d_ad, d_x + 16, y + 4 * at, res=res + 4 * at, x_stride=x_stride,
                                    y_stride=y_stride), box.dev.last_error()
        got = box.down(y, wide).reshape(-1)
        beside = np.ones(got.size, bool)
        for t in range(tokens):
            s = slice(at + t * y_stride, at + t * y_stride + rows)
            check(got[s], want[t], bound[t])
            beside[s] = False
        assert (got[beside] == (flat[beside] if y == d_res else 7)).all()


def test_what_is_not_a_number_stays_with_its_token(box):
    rng = np.random.default_rng(8)
    c = Case(zd.BF16, 40, 4, 16, 70, 64, rng, np.arange(40) % 3)
    c.x[5, 9], c.x[7, 3], c.res[9, 4] = np.nan, np.inf, np.inf
    c.a[3], c.b[3] = 0x7FC0, 0x7FC0  # an adapter that no token has
    got = run(box, c)
    assert np.isnan(got[5]).all() and np.isnan(got[7]).all() and np.isinf(got[9, 4])
    c.x[[5, 7]] = 0
    want, bound = c.want()
    want[9, 4] = bound[9, 4] = 0
    rest = [t for t in range(40) if t not in (5, 7)]
    got[9, 4] = 0
    check(got[rest], want[rest], bound[rest])


@pytest.mark.parametrize("tokens", [6, 150, 400, 1300])
def test_captured(box, tokens):
    """Two graphs over one scratch, replayed for other adapters, tokens and residuals, against eager calls."""
    dev = box.dev
    _say(f"lora graph tokens={tokens}")
    rng = np.random.default_rng(9)
    c = Case(zd.F16, tokens, 6, 32, 200, 512, rng)
    lora, d_ad, d_x, d_res = c.up(box), box.up(c.adapter), box.up(c.x), box.up(c.res)
    outs = [box.up(np.zeros_like(c.res)) for _ in range(3)]

    def step(y):
        assert dev.lora_enqueue(lora, tokens, d_ad, d_x, y, res=d_res), dev.last_error()

    step(outs[2])
    graphs = []
    for y in outs[:2]:
        assert dev.capture_begin(), dev.last_error()
        step(y)
        graphs.append(dev.capture_end())
        assert graphs[-1], dev.last_error()
    try:
        for _ in range(3):
            c.adapter = rng.integers(-1, 6, tokens).astype(np.int32)
            c.x = rng.standard_normal(c.x.shape).astype(np.float32)
            dev.dev_upload(d_ad, c.adapter)
            dev.dev_upload(d_x, c.x)
            want, bound = c.want()
            got = []
            for g, y in zip(graphs, outs):
                dev.dev_upload(y, np.full_like(c.res, 9))
                dev.graph_launch(g, 2)
                got.append(box.down(y, c.res))
                step(outs[2])
            got.append(box.down(outs[2], c.res))
            check(got[2], want, bound)
            np.testing.assert_array_equal(got[0], got[2])
            np.testing.assert_array_equal(got[1], got[2])
    finally:
        for g in graphs:
            dev.graph_destroy(g)


def test_pools_past_32_bits(box):
    """An adapter whose A and B lie more than 2^32 bytes into their pools."""
    n, rank, rows, k = 1100, 256, 9000, 8192
    _say("lora far pools")
    rng = np.random.default_rng(10)
    small = Case(zd.F16, 3, 1, rank, rows, k, rng, [0, 0, -1])
    size_a, size_b = 2 * rank * k, 2 * rank * rows
    assert size_a * (n - 1) > 1 << 32 and size_b * (n - 1) > 1 << 32
    d_a, d_b = box.dev.dev_malloc(n * size_a), box.dev.dev_malloc(n * size_b)
    box.bufs += [d_a, d_b]
    box.dev.dev_upload(d_a + (n - 1) * size_a, small.a)
    box.dev.dev_upload(d_b + (n - 1) * size_b, small.b)
    lora = zd.Lora(d_a, d_b, zd.F16, n, rank, rows, k)
    d_y = box.up(small.res)
    assert box.dev.lora_enqueue(lora, 3, box.up(np.array([n - 1, n - 1, n], np.int32)), box.up(small.x), d_y, res=d_y), \
        box.dev.last_error()
    check(box.down(d_y, small.res), *small.want())
