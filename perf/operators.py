"""The serving operators over a paged KV cache, and the sampler, as measurable cases.

Kinds:

* ``append``  q/k head norm, rotary embedding and the append of K and V of a batch of
  tokens to a paged cache (f16, or 4-bit q4_0 blocks); returns the rotated q and what
  the cache holds now: the f16 pages, or the 4-bit rows of the batch as the values they
  stand for (read back from the cache);
* ``attend``  attention of a batch of tokens over the paged cache: one token a sequence
  (decode), a few (verification), many (a prompt's chunk), or both in one batch;
* ``sample``  one token a row of logits by temperature, top-k, top-p and min-p from a
  given uniform number, and its probability among the tokens kept.

A page holds ``page`` positions of every kv head; K and V have a pool each.  Per head:

* K: f16 [page][hd]; q4_0: [page][hd/32][16 bytes] (the nibbles of a GGUF q4_0 block),
  then the f16 scales [page][hd/32];
* V, in groups of 8 positions: f16 [page/8][hd][8]; q4_0: one 32-bit word of 8 nibbles
  per (group, dim), position j's at bits 4*(j/2) + 16*(j%2), [page/8][hd], then the f16
  scales [page/8][hd/32][8].

A q4_0 value is d * (nibble - 8), d an f16 of at most 8 significant bits.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
_dev = None


def listed():
    return [
        # one token of an 8B model (32 q / 8 kv heads of 128) to an f16 cache: the smallest call, once a layer and token
        {"name": "append_1_f16", "kind": "append", "cache": "f16", "heads": 32, "kv": 8, "hd": 128, "page": 64,
         "seqs": 1, "prefill": 0, "q_max": 1, "kv_max": 2048, "spread": 0.0, "norm": True, "base": 1e6},
        # 64 sequences' next tokens to a 4-bit cache, positions up to 100000
        {"name": "append_64_q4", "kind": "append", "cache": "q4_0", "heads": 32, "kv": 8, "hd": 128, "page": 64,
         "seqs": 64, "prefill": 0, "q_max": 1, "kv_max": 100000, "spread": 0.9, "norm": True, "base": 1e6},
        # two prompts' chunks to a 4-bit cache, ragged
        {"name": "append_prompts_q4", "kind": "append", "cache": "q4_0", "heads": 32, "kv": 8, "hd": 128, "page": 64,
         "seqs": 2, "prefill": 2, "q_max": 4099, "kv_max": 9001, "spread": 0.3, "norm": True, "base": 1e6},
        # one token over 2048 cached positions, 4 bits
        {"name": "decode_1_q4", "kind": "attend", "cache": "q4_0", "heads": 32, "kv": 8, "hd": 128, "page": 64,
         "seqs": 1, "prefill": 0, "q_max": 1, "kv_max": 2048, "spread": 0.0, "window": 0},
        # a serving batch: 64 sequences of 820 to 8192 positions, 4 bits
        {"name": "decode_64_q4", "kind": "attend", "cache": "q4_0", "heads": 32, "kv": 8, "hd": 128, "page": 64,
         "seqs": 64, "prefill": 0, "q_max": 1, "kv_max": 8192, "spread": 0.9, "window": 0},
        # few long f16 sequences in pages of 16
        {"name": "decode_6_long_f16", "kind": "attend", "cache": "f16", "heads": 32, "kv": 8, "hd": 128, "page": 16,
         "seqs": 6, "prefill": 0, "q_max": 1, "kv_max": 32001, "spread": 0.8, "window": 0},
        # verification of 5 drafted tokens in 8 sequences, 4 bits
        {"name": "verify_8x5_q4", "kind": "attend", "cache": "q4_0", "heads": 32, "kv": 8, "hd": 128, "page": 64,
         "seqs": 8, "prefill": 8, "q_max": 5, "kv_max": 4000, "spread": 0.5, "window": 0},
        # a prompt's chunk of 2048 tokens that ends at position 7999, 4 bits
        {"name": "chunk_2048_q4", "kind": "attend", "cache": "q4_0", "heads": 32, "kv": 8, "hd": 128, "page": 64,
         "seqs": 1, "prefill": 1, "q_max": 2048, "kv_max": 8000, "spread": 0.0, "window": 0},
        # a prompt of 1000 tokens beside 15 decoding sequences, heads of 256 with a window, f16
        {"name": "mixed_16_window_f16", "kind": "attend", "cache": "f16", "heads": 16, "kv": 8, "hd": 256, "page": 32,
         "seqs": 16, "prefill": 1, "q_max": 1000, "kv_max": 3000, "spread": 0.7, "window": 1024},
        # one row of a 151936-token vocabulary: the end of every token at batch 1
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": 151936, "top_k": 50, "top_p": 0.95, "min_p": 0.0,
         "greedy": 0.0, "masked": 0.0, "std": 2.5},
        # 64 rows, nucleus only, a tenth of the rows greedy
        {"name": "sample_64_top_p", "kind": "sample", "rows": 64, "vocab": 128256, "top_k": 0, "top_p": 0.9,
         "min_p": 0.0, "greedy": 0.1, "masked": 0.0, "std": 2.5},
        # 256 rows of the largest vocabulary at temperature alone with a min-p, half the tokens masked by a grammar
        {"name": "sample_256_min_p", "kind": "sample", "rows": 256, "vocab": 262144, "top_k": 0, "top_p": 1.0,
         "min_p": 0.02, "greedy": 0.0, "masked": 0.5, "std": 2.5},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "sample", "sample"])
    if kind == "sample":
        vocab = _log(rng, 1000, 262144)
        k = rng.choice([0, 0, 1, 50, _log(rng, 2, 2000)])
        return {"kind": kind, "rows": max(1, min(_log(rng, 1, 256), 256 * 262144 // vocab)), "vocab": vocab,
                "top_k": k, "top_p": rng.choice([1.0, round(rng.uniform(0.05, 0.999), 3)]),
                "min_p": rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]), "greedy": rng.choice([0.0, 0.2]),
                "masked": rng.choice([0.0, 0.5, 0.95]), "std": round(rng.uniform(0.3, 4.0), 2)}
    kv = rng.choice([1, 2, 4, 8])
    hd = rng.choice([64, 128, 128, 256])
    c = {"kind": kind, "cache": rng.choice(["f16", "q4_0"]), "heads": kv * rng.choice([1, 2, 3, 4, 5, 8]), "kv": kv,
         "hd": hd, "page": rng.choice([16, 32, 64, 128, 256])}
    shape = rng.choice(["decode", "decode", "few", "prompt", "mixed"])
    if kind == "append":
        seqs = _log(rng, 1, 256) if shape in ("decode", "few") else rng.randint(1, 8)
        q_max = {"decode": 1, "few": rng.randint(2, 8)}.get(shape) or _log(rng, 33, 4096)
        q_max = max(1, min(q_max, 8192 * 48 * 128 // ((c["heads"] + 2 * kv) * hd * seqs)))
        c.update(seqs=seqs, prefill=0 if shape == "decode" else 1 if shape == "mixed" else seqs, q_max=q_max,
                 kv_max=max(q_max, _log(rng, 1, 200000)), spread=round(rng.uniform(0, 0.95), 2),
                 norm=rng.random() < 0.7, base=rng.choice([1e4, 5e5, 1e6]))
        return c
    seqs = _log(rng, 1, 64) if shape in ("decode", "few") else rng.randint(1, 12)
    q_max = {"decode": 1, "few": rng.randint(2, 8)}.get(shape) or _log(rng, 33, 2048)
    kv_max = max(q_max, _log(rng, 1, 32000))
    # at most 64 sequences of 8192 positions and 8 kv heads of 128, and the flops of the longest chunk
    kv_max = max(q_max, min(kv_max, 64 * 8192 * 8 * 128 // (seqs * kv * hd)))
    n_pre = 0 if shape == "decode" else 1 if shape == "mixed" else seqs
    while n_pre and n_pre * q_max * kv_max * c["heads"] * hd > 2048 * 8000 * 32 * 128:
        q_max = max(1, q_max // 2)
        kv_max = max(q_max, kv_max * 2 // 3)
    # the plain form pads every sequence to the longest: its scores stay within 8 GB
    while seqs > 1 and seqs * q_max * kv_max * c["heads"] > 2_000_000_000:
        seqs = max(1, seqs // 2)
        n_pre = min(n_pre, seqs)
    c.update(seqs=seqs, prefill=n_pre, q_max=q_max, kv_max=kv_max, spread=round(rng.uniform(0, 0.95), 2),
             window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]))
    return c


# ---- sizes of a case ------------------------------------------------------------------


def _lens(c):
    """(tokens, cached positions with them) of every sequence: the prompts first, lengths spread below the largest."""
    q, kv = [], []
    for i in range(c["seqs"]):
        n = max(1, round(c["q_max"] * (1 - 0.3 * ((i * 0.7548776662) % 1)))) if i < c["prefill"] else 1
        q.append(n)
        kv.append(max(n, round(c["kv_max"] * (1 - c["spread"] * ((i * 0.6180339887) % 1)))))
    return q, kv


def _row_bytes(c):
    return c["hd"] * 2 if c["cache"] == "f16" else c["hd"] // 2 + c["hd"] // 16


# ---- inputs ---------------------------------------------------------------------------


class _Inputs:
    """The seeded stream of a case: the same tensors in the same order for prepare() and exact()."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda", dtype=torch.float32)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.gen, device="cuda", dtype=torch.float32)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pages(c, g):
    """(table of pages, pages): every sequence's pages scattered over the pool.  An append's table names the pages
    that it writes only; -1 stands where a sequence has none."""
    q, kv = _lens(c)
    page = c["page"]
    first = [(n - t) // page if c["kind"] == "append" else 0 for t, n in zip(q, kv)]
    last = [(n + page - 1) // page for n in kv]
    total = sum(b - a for a, b in zip(first, last))
    order = g.order(total).to(torch.int32).cpu()
    table = torch.full((c["seqs"], max(last)), -1, dtype=torch.int32)
    at = 0
    for i, (a, b) in enumerate(zip(first, last)):
        table[i, a:b] = order[at:at + b - a]
        at += b - a
    return table.cuda(), total


def _cache_values(c, g, pages):
    """What an attention's cache holds, by position: K and V of every page as (values f16) or (nibbles u8, scales f16),
    each [pages, kv, page, hd] (scales [pages, kv, page, hd/32])."""
    shape = (pages, c["kv"], c["page"], c["hd"])
    got = []
    for _ in range(2):
        x = g.normal(*shape)
        if c["cache"] == "f16":
            got.append((x.half(), None))
        else:
            n = (x * 2.8 + 8.5).floor_().clamp_(0, 15).to(torch.uint8)
            d = (0.3 * (1 + 0.1 * g.normal(*shape[:3], shape[3] // 32))).bfloat16().half()
            got.append((n, d))
    return got


def _pack_k(c, v, d):
    """K's pool, bytes [pages, kv, page * row bytes]."""
    p = v.shape[0]
    if d is None:
        return v.reshape(p, c["kv"], -1).view(torch.uint8).clone()
    b = v.reshape(p, c["kv"], c["page"], c["hd"] // 32, 2, 16)
    nib = (b[..., 0, :] | (b[..., 1, :] << 4)).reshape(p, c["kv"], -1)
    return torch.cat([nib, d.reshape(p, c["kv"], -1).view(torch.uint8)], 2)


def _pack_v(c, v, d):
    """V's pool, bytes [pages, kv, page * row bytes]."""
    p, groups = v.shape[0], c["page"] // 8
    if d is None:
        return v.reshape(p, c["kv"], groups, 8, c["hd"]).transpose(3, 4).reshape(p, c["kv"], -1).view(torch.uint8)
    b = v.reshape(p, c["kv"], groups, 4, 2, c["hd"])  # positions 2i and 2i + 1
    halves = [sum(b[..., i, h, :].to(torch.int32) << (4 * i) for i in range(4)) for h in range(2)]
    words = (halves[0] | (halves[1] << 16)).reshape(p, c["kv"], -1)
    s = d.reshape(p, c["kv"], groups, 8, c["hd"] // 32).transpose(3, 4).reshape(p, c["kv"], -1)
    return torch.cat([words.view(torch.uint8), s.view(torch.uint8)], 2)


class _State:
    pass


def _logits(c, g):
    """Rows as a model gives them: a bell, a few tokens that stand out, and the tokens that a grammar forbids."""
    x = c["std"] * g.normal(c["rows"], c["vocab"])
    lead = (torch.arange(8, device="cuda") * 0.6180339887 * c["vocab"]).long() % c["vocab"]
    x[:, lead] += 2.0 * c["std"]
    if c["masked"]:
        keep = g.uniform(c["rows"], c["vocab"]) >= c["masked"]
        keep[:, 7 % c["vocab"]] = True
        x.masked_fill_(~keep, -math.inf)
    return x


def _params(c, g):
    """(temperature, top-k, top-p, min-p, uniform numbers) of every row; temperature 0 is greedy."""
    r = c["rows"]
    t = 0.5 + g.uniform(r)
    t[g.uniform(r) < c["greedy"]] = 0.0
    full = lambda v, kind: torch.full((r,), v, dtype=kind, device="cuda")  # noqa: E731
    return (t, full(c["top_k"], torch.int32), full(c["top_p"], torch.float32), full(c["min_p"], torch.float32),
            g.uniform(r))


def _append_inputs(c, g):
    q, kv = _lens(c)
    table, pages = _pages(c, g)
    qkv = g.normal(sum(q), (c["heads"] + 2 * c["kv"]) * c["hd"])
    qn, kn = 1 + 0.1 * g.normal(c["hd"]), 1 + 0.1 * g.normal(c["hd"])
    return q, kv, table, pages, qkv, qn, kn


def _attend_inputs(c, g):
    q, kv = _lens(c)
    table, pages = _pages(c, g)
    x = 1.5 * g.normal(sum(q), c["heads"], c["hd"])
    return q, kv, table, pages, x, _cache_values(c, g, pages)


def _starts(q):
    at = [0]
    for n in q:
        at.append(at[-1] + n)
    return at


def prepare(case, seed):
    c, g, s = case, _Inputs(seed), _State()
    s.case = c
    if c["kind"] == "sample":
        s.logits = _logits(c, g)
        s.temperature, s.top_k, s.top_p, s.min_p, s.u = _params(c, g)
        s.token = torch.empty(c["rows"], dtype=torch.int32, device="cuda")
        s.prob = torch.empty(c["rows"], device="cuda")
        torch.cuda.synchronize()  # the backend has a stream of its own
        return s
    if c["kind"] == "append":
        q, kv, s.table, s.pages, s.qkv, s.qn, s.kn = _append_inputs(c, g)
        size = (s.pages, c["kv"], c["page"] * _row_bytes(c))
        s.k_pool, s.v_pool = (torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(2))
        s.q_out = torch.empty(sum(q), c["heads"], c["hd"], device="cuda")
        s.k_out, s.v_out = (torch.empty(sum(q), c["kv"], c["hd"], device="cuda") for _ in range(2))
    else:
        q, kv, s.table, s.pages, s.q, (k, v) = _attend_inputs(c, g)
        s.k_pool, s.v_pool = _pack_k(c, *k), _pack_v(c, *v)
        s.out = torch.empty_like(s.q)
    s.tokens, s.longest, s.deepest = sum(q), max(q), max(kv)
    s.q_start, s.kv_len = _ints(_starts(q)), _ints(kv)
    torch.cuda.synchronize()  # the backend has a stream of its own
    return s


# ---- one pass: the framework's calls -----------------------------------------------------


def _device():
    from zlm_amd import device as zd
    global _dev
    if _dev is None:
        _dev = zd.Device()
        if not _dev.available():
            raise RuntimeError(_dev.last_error())
    return zd, _dev


def _run_own(s):
    zd, d = _device()
    c = s.case
    if c["kind"] == "sample":
        ok = d.sample_enqueue(s.logits.data_ptr(), c["rows"], c["vocab"], s.u.data_ptr(), s.token.data_ptr(),
                              temperature=s.temperature.data_ptr(), top_k=s.top_k.data_ptr(),
                              top_p=s.top_p.data_ptr(), min_p=s.min_p.data_ptr(), prob=s.prob.data_ptr())
        if not ok:
            raise RuntimeError(d.last_error())
        return {"token": s.token, "prob": s.prob}
    kind = zd.F16 if c["cache"] == "f16" else zd.Q4_0
    cache = zd.PagedCache(s.k_pool.data_ptr(), s.v_pool.data_ptr(), kind, c["kv"], c["hd"], c["page"], s.pages)
    batch = zd.PagedBatch(c["seqs"], s.tokens, s.q_start.data_ptr(), s.kv_len.data_ptr(), s.table.data_ptr(),
                          s.table.shape[1])
    if c["kind"] == "attend":
        if not d.paged_attention_enqueue(cache, batch, s.q.data_ptr(), s.out.data_ptr(), c["heads"],
                                         c["hd"] ** -0.5, window=c["window"]):
            raise RuntimeError(d.last_error())
        return s.out
    norm = (s.qn.data_ptr(), s.kn.data_ptr()) if c["norm"] else (0, 0)
    if not d.paged_append_enqueue(cache, batch, s.qkv.data_ptr(), s.q_out.data_ptr(), c["heads"], EPS, c["base"],
                                  q_norm_w=norm[0], k_norm_w=norm[1]):
        raise RuntimeError(d.last_error())
    if c["cache"] == "f16":
        return {"q": s.q_out, "k": s.k_pool.view(torch.float16), "v": s.v_pool.view(torch.float16)}
    if not d.paged_read_enqueue(cache, batch, s.k_out.data_ptr(), s.v_out.data_ptr()):
        raise RuntimeError(d.last_error())
    return {"q": s.q_out, "k": s.k_out, "v": s.v_out}


# ---- one pass: the plain form -------------------------------------------------------------


def _token_places(s):
    """(sequence, position) of every token of the batch."""
    t = torch.arange(s.tokens, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s.q_start[1:].contiguous(), t, right=True)
    pos = s.kv_len[seq] - (s.q_start[seq + 1] - s.q_start[seq]) + (t - s.q_start[seq])
    return seq, pos.long()


def _quantise(x):
    """(nibbles, scales) of the q4_0 blocks of x (float64, [..., hd])."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    at = b.abs().argmax(-1, keepdim=True)  # the first of the largest
    m = torch.gather(b, -1, at)[..., 0]
    d = (m / -8).float().bfloat16().float().clamp(-2720, 2720).half()
    dd = d.double()[..., None]
    n = torch.where(dd != 0, torch.floor(b / torch.where(dd != 0, dd, 1.0) + 8.5), 8.0).clamp(0, 15)
    return n.to(torch.int32).reshape(x.shape), d


def _rotated(s, x, w, pos):
    """x (float64, [tokens, heads, hd]): head norm, then the rotation by the position."""
    c = s.case
    if c["norm"]:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    half = c["hd"] // 2
    inv = torch.pow(torch.tensor(c["base"], dtype=torch.float64, device="cuda"),
                    torch.arange(half, dtype=torch.float64, device="cuda") * (-2.0 / c["hd"]))
    a = (pos.double()[:, None] * inv)[:, None, :]
    cos, sin = a.cos(), a.sin()
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], -1)


def _append_plain(s):
    c = s.case
    kv, hd, page = c["kv"], c["hd"], c["page"]
    seq, pos = _token_places(s)
    x = s.qkv.double().reshape(s.tokens, -1, hd)
    q = _rotated(s, x[:, :c["heads"]], s.qn, pos).float()
    k, v = _rotated(s, x[:, c["heads"]:c["heads"] + kv], s.kn, pos), x[:, c["heads"] + kv:]
    p, off = s.table[seq, pos // page].long(), pos % page
    if c["cache"] == "f16":
        kp = s.k_pool.view(torch.float16).view(s.pages, kv, page, hd)
        vp = s.v_pool.view(torch.float16).view(s.pages, kv, page // 8, hd, 8)
        kp[p, :, off] = k.half()
        vp[p, :, off // 8, :, off % 8] = v.half()
        return {"q": q, "k": s.k_pool.view(torch.float16), "v": s.v_pool.view(torch.float16)}
    nibbles = page * hd // 2
    (kn, kd), (vn, vd) = _quantise(k), _quantise(v)
    b = kn.reshape(s.tokens, kv, hd // 32, 2, 16)
    s.k_pool[:, :, :nibbles].view(s.pages, kv, page, hd // 2)[p, :, off] = \
        (b[..., 0, :] | (b[..., 1, :] << 4)).to(torch.uint8).reshape(s.tokens, kv, -1)
    s.k_pool[:, :, nibbles:].view(torch.float16).view(s.pages, kv, page, hd // 32)[p, :, off] = kd
    words = s.v_pool.view(torch.int32)[:, :, :page * hd // 8].view(s.pages, kv, page // 8, hd)
    heads, dims = torch.arange(kv, device="cuda")[None, :, None], torch.arange(hd, device="cuda")[None, None, :]
    place = (p[:, None, None], heads, (off // 8)[:, None, None], dims)
    shift = (4 * (off % 8 // 2) + 16 * (off % 2)).to(torch.int32)[:, None, None]
    old = (words[place] >> shift) & 15
    words.index_put_(place, (vn - old) << shift, accumulate=True)  # a nibble's change; its neighbours keep theirs
    scales = s.v_pool[:, :, nibbles:].view(torch.float16).view(s.pages, kv, page // 8, hd // 32, 8)
    scales[p, :, off // 8, :, off % 8] = vd
    # the rows as the cache holds them now
    kb = s.k_pool[:, :, :nibbles].view(s.pages, kv, page, hd // 32, 16)[p, :, off].to(torch.int32)
    kd = s.k_pool[:, :, nibbles:].view(torch.float16).view(s.pages, kv, page, hd // 32)[p, :, off]
    vw = (words[place] >> shift) & 15
    vd = scales[p, :, off // 8, :, off % 8]
    k = (torch.cat([kb & 15, kb >> 4], -1) - 8) * kd.float()[..., None]
    v = (vw.reshape(s.tokens, kv, hd // 32, 32) - 8) * vd.float()[..., None]
    return {"q": q, "k": k.reshape(s.tokens, kv, hd), "v": v.reshape(s.tokens, kv, hd)}


def _cached(s):
    """K and V of every sequence, float32 [seqs, kv, positions, hd], from the pages."""
    c = s.case
    kv, hd, page = c["kv"], c["hd"], c["page"]
    used = s.table.long().clamp_min(0)
    n, per = used.shape
    k, v = s.k_pool[used], s.v_pool[used]  # [seqs, pages, kv, bytes]
    if c["cache"] == "f16":
        k = k.view(torch.float16).view(n, per, kv, page, hd).float()
        v = v.view(torch.float16).view(n, per, kv, page // 8, hd, 8).transpose(4, 5).reshape(n, per, kv, page, hd)
        v = v.float()
    else:
        nib = page * hd // 2
        b = k[..., :nib].reshape(n, per, kv, page, hd // 32, 16)
        d = k[..., nib:].contiguous().view(torch.float16).view(n, per, kv, page, hd // 32, 1).float()
        k = ((torch.cat([b & 15, b >> 4], -1).float() - 8) * d).reshape(n, per, kv, page, hd)
        w = v[..., :nib].contiguous().view(torch.int32).view(n, per, kv, page // 8, hd, 1)
        j = torch.arange(8, device="cuda", dtype=torch.int32)
        w = ((w >> (4 * (j // 2) + 16 * (j % 2))) & 15).to(torch.uint8)
        d = v[..., nib:].contiguous().view(torch.float16).view(n, per, kv, page // 8, hd // 32, 1, 8).float()
        v = (w.view(n, per, kv, page // 8, hd // 32, 32, 8).float() - 8) * d
        v = v.view(n, per, kv, page // 8, hd, 8).transpose(4, 5).reshape(n, per, kv, page, hd)
    join = lambda x: x.permute(0, 2, 1, 3, 4).reshape(n, kv, per * page, hd)[:, :, :s.deepest].contiguous()  # noqa: E731
    return join(k), join(v)


def _attend_plain(s):
    c = s.case
    kv, hd, g = c["kv"], c["hd"], c["heads"] // c["kv"]
    seq, pos = _token_places(s)
    k, v = _cached(s)
    n = c["seqs"]
    row = torch.arange(s.tokens, device="cuda") - s.q_start[seq]
    q = torch.zeros(n, s.longest, kv, g, hd, device="cuda")
    q[seq, row] = s.q.view(s.tokens, kv, g, hd)
    q = q.permute(0, 2, 1, 3, 4).reshape(n * kv, s.longest * g, hd)
    at = torch.full((n, s.longest), -1, dtype=torch.long, device="cuda")
    at[seq, row] = pos
    j = torch.arange(s.deepest, device="cuda")
    seen = (j <= at[..., None]) & ((j > at[..., None] - c["window"]) if c["window"] else True)
    scores = torch.bmm(q * hd ** -0.5, k.view(n * kv, -1, hd).transpose(1, 2).contiguous())
    scores = scores.view(n, kv, s.longest, g, -1).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.bmm(scores.view(n * kv, s.longest * g, -1), v.view(n * kv, -1, hd))
    out = out.view(n, kv, s.longest, g, hd) / total
    return out.permute(0, 2, 1, 3, 4)[seq, row].reshape(s.tokens, c["heads"], hd)


def _sample_plain(s):
    x, at = torch.sort(s.logits, dim=1, descending=True, stable=True)
    rank = torch.arange(x.shape[1], device="cuda")
    t = s.temperature.double()[:, None]
    x = x.double()
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    k = s.top_k.long()[:, None]
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    run_up = w.cumsum(1)
    w = torch.where(run_up - w < s.top_p.double()[:, None] * run_up[:, -1:], w, 0.0)
    w = torch.where(w >= s.min_p.double()[:, None], w, 0.0)
    w = torch.where((t > 0) | (rank < 1), w, 0.0)  # temperature 0: the largest
    run_up = w.cumsum(1)
    total = run_up[:, -1:]
    first = (run_up <= s.u.double()[:, None] * total).sum(1, keepdim=True)
    prob = torch.gather(w, 1, first) / total
    return {"token": torch.gather(at, 1, first)[:, 0].int(), "prob": prob[:, 0].float()}


def run(state):
    if own:
        return _run_own(state)
    return {"append": _append_plain, "attend": _attend_plain, "sample": _sample_plain}[state.case["kind"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    c = case
    if c["kind"] == "sample":
        return {"bytes": c["rows"] * (4 * c["vocab"] + 28), "flops": 8 * c["rows"] * c["vocab"]}
    q, kv = _lens(c)
    tokens, head = sum(q), c["kv"] * c["hd"]
    table = 4 * sum((n + c["page"] - 1) // c["page"] for n in kv)
    if c["kind"] == "append":
        values = 0 if c["cache"] == "f16" else 8 * head
        return {"bytes": tokens * (8 * c["heads"] * c["hd"] + 8 * head + 2 * c["kv"] * _row_bytes(c) + values)
                + 8 * c["seqs"], "flops": tokens * 12 * (c["heads"] + 2 * c["kv"]) * c["hd"]}
    cached = pairs = 0
    for n, end in zip(q, kv):
        w = c["window"] or end
        cached += end - max(0, end - n + 1 - w)
        pairs += sum(min(p + 1, w) for p in range(end - n, end))
    return {"bytes": 2 * cached * c["kv"] * _row_bytes(c) + 8 * tokens * c["heads"] * c["hd"] + table,
            "flops": 4 * pairs * c["heads"] * c["hd"]}


# ---- the same in 64 bits, from the definitions ------------------------------------------------


def _spot(c, table, i, p):
    """(page, offset) of position p of sequence i."""
    return int(table[i, p // c["page"]]), p % c["page"]


def _rope64(x, base, pos):
    """x [n, heads, hd] float64 as complex pairs (i, i + hd/2) turned by pos * base^(-2i/hd)."""
    n = x.shape[-1] // 2
    i = torch.arange(n, dtype=torch.float64, device=x.device)
    turn = torch.exp(i * (-2.0 / x.shape[-1]) * math.log(base))[None, :] * pos[:, None]
    z = torch.complex(x[..., :n], x[..., n:]) * torch.polar(torch.ones_like(turn), turn)[:, None, :]
    return torch.cat([z.real, z.imag], -1)


def _q4_values(x):
    """The values that q4_0 blocks hold for x (float64)."""
    b = x.reshape(-1, 32)
    lo, hi = b.min(1), b.max(1)
    tie = torch.gather(b, 1, torch.minimum(lo.indices, hi.indices)[:, None])[:, 0]
    big = torch.where(-lo.values > hi.values, lo.values, torch.where(-lo.values < hi.values, hi.values, tie))
    d = (big / -8).to(torch.float32).to(torch.bfloat16).to(torch.float16).double()[:, None]
    n = torch.floor(b / d.masked_fill(d == 0, 1.0) + 8.5).clamp(0, 15)
    return ((n - 8) * d).reshape(x.shape)


def _append_exact(c, g):
    q, kv, table, pages, qkv, qn, kn = _append_inputs(c, g)
    x = qkv.double().reshape(sum(q), -1, c["hd"])
    where = [(i, p) for i, (n, end) in enumerate(zip(q, kv)) for p in range(end - n, end)]
    pos = torch.tensor([p for _, p in where], dtype=torch.float64, device="cuda")

    def head(y, w):
        if c["norm"]:
            y = y * torch.rsqrt(y.pow(2).sum(-1, keepdim=True) / c["hd"] + EPS) * w.double()
        return _rope64(y, c["base"], pos)

    h = c["heads"]
    got = {"q": head(x[:, :h], qn), "k": head(x[:, h:h + c["kv"]], kn), "v": x[:, h + c["kv"]:]}
    if c["cache"] == "q4_0":
        return {"q": got["q"], "k": _q4_values(got["k"].contiguous()), "v": _q4_values(got["v"].contiguous())}
    table = table.cpu()
    spots = torch.tensor([_spot(c, table, i, p) for i, p in where], device="cuda")
    pools = {}
    for name in ("k", "v"):
        pool = torch.zeros(pages, c["kv"], c["page"], c["hd"], dtype=torch.float64, device="cuda")
        pool[spots[:, 0], :, spots[:, 1]] = got[name]
        pools[name] = pool
    v = pools["v"].unflatten(2, (-1, 8)).transpose(3, 4)
    return {"q": got["q"], "k": pools["k"].reshape(pages, c["kv"], -1), "v": v.reshape(pages, c["kv"], -1)}


def _attend_exact(c, g):
    q, kv, table, _, x, (k, v) = _attend_inputs(c, g)
    table = table.long()
    out, at, group = [], 0, c["heads"] // c["kv"]

    def rows(values, scales, pages):
        y = values[pages].double()
        if scales is not None:
            y = (y.unflatten(-1, (-1, 32)) - 8) * scales[pages].double().unsqueeze(-1)
            y = y.flatten(-2)
        return y.transpose(0, 1).flatten(1, 2)  # [kv, positions, hd]

    for i, (n, end) in enumerate(zip(q, kv)):
        pages = table[i, :(end + c["page"] - 1) // c["page"]]
        kk, vv = (rows(*t, pages)[:, :end] for t in (k, v))
        p = torch.arange(end - n, end, device="cuda")[:, None]
        j = torch.arange(end, device="cuda")[None, :]
        off = (j > p) | (j <= p - c["window"] if c["window"] else j > p)
        heads = []
        for h in range(c["heads"]):
            score = x[at:at + n, h].double() @ kk[h // group].T.contiguous() / math.sqrt(c["hd"])
            heads.append(torch.softmax(score.masked_fill(off, -math.inf), 1) @ vv[h // group])
        out.append(torch.stack(heads, 1))
        at += n
    return torch.cat(out)


def _sample_exact(c, g):
    logits = _logits(c, g)
    temperature, top_k, top_p, min_p, u = (t.tolist() for t in _params(c, g))
    tokens, probs = [], []
    for r in range(c["rows"]):
        x = logits[r].double()
        if temperature[r] <= 0:
            tokens.append(int(x.argmax()))
            probs.append(1.0)
            continue
        order = torch.argsort(-x, stable=True)
        if 0 < top_k[r]:
            order = order[:top_k[r]]
        p = torch.softmax(x[order] / temperature[r], 0)
        before = torch.cat([p.new_zeros(1), p.cumsum(0)[:-1]])
        keep = (before < top_p[r]) & (p >= min_p[r] * p[0])
        order, p = order[keep], p[keep] / p[keep].sum()
        at = min(int((p.cumsum(0) <= u[r]).sum()), len(p) - 1)
        tokens.append(int(order[at]))
        probs.append(float(p[at]))
    return {"token": torch.tensor(tokens, dtype=torch.int32), "prob": torch.tensor(probs, dtype=torch.float64)}


def exact(case, seed):
    return {"append": _append_exact, "attend": _attend_exact, "sample": _sample_exact}[case["kind"]](case, _Inputs(seed))
