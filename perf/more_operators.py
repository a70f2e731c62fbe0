"""Further serving operators, as measurable cases.

Kinds:

* ``append``  q/k head norm, rotary embedding and the append of a batch's K and V to a paged cache
  of 8-bit numbers (e4m3) with a scale for each 16 positions and head; returns the rotated q, and
  what the cache holds now of the blocks that the batch wrote (its own rows and those before them
  in a block that it found begun, whose scale it may have raised);
* ``attend``  attention of a batch over that cache, or over any paged cache (f16, q4_0, e4m3) by a
  sliding window beside a few first positions that stay visible;
* ``verify``  drafted tokens against a target's logits from given random numbers: how many are
  accepted, and the token drawn after them, so that every token has the target's distribution;
* ``lora``    low-rank adapters of many requests beside a shared projection,
  y = res + scale * B (A x) with each token's own A, B and scale.

Pages of an e4m3 cache, per head: K [page][hd] bytes, V [page/8][hd][8] bytes, each followed by 16
bytes, of which the first page/16 are the blocks' scales, 2^(byte - 127) with byte 112 to 134.
Those of the other caches are as ``operators.py`` beside this says.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
K_MIN, K_MAX = -15, 7  # of a block's scale, 2^k
_dev = None


def listed():
    return [
        # one token of an 8B model (32 q / 8 kv heads of 128), in the middle of a block: once a layer and token
        {"name": "append_1", "kind": "append", "heads": 32, "kv": 8, "hd": 128, "page": 64, "seqs": 1, "prefill": 0,
         "q_max": 1, "kv_max": 2043, "spread": 0.0, "norm": True, "base": 1e6},
        # two prompts' chunks, ragged, that begin inside blocks
        {"name": "append_prompts", "kind": "append", "heads": 32, "kv": 8, "hd": 128, "page": 64, "seqs": 2,
         "prefill": 2, "q_max": 4099, "kv_max": 9001, "spread": 0.3, "norm": True, "base": 1e6},
        # a serving batch over the 8-bit cache: 64 sequences of 820 to 8192 positions
        {"name": "decode_64", "kind": "attend", "cache": "e4m3", "heads": 32, "kv": 8, "hd": 128, "page": 64,
         "seqs": 64, "prefill": 0, "q_max": 1, "kv_max": 8192, "spread": 0.9, "window": 0, "sinks": 0},
        # a prompt's chunk of 2048 tokens that ends at position 7999 of the 8-bit cache
        {"name": "chunk_2048", "kind": "attend", "cache": "e4m3", "heads": 32, "kv": 8, "hd": 128, "page": 64,
         "seqs": 1, "prefill": 1, "q_max": 2048, "kv_max": 8000, "spread": 0.0, "window": 0, "sinks": 0},
        # one endless stream: 4 sinks and the last 1020 positions, 8 bits
        {"name": "stream_1", "kind": "attend", "cache": "e4m3", "heads": 32, "kv": 8, "hd": 128, "page": 64,
         "seqs": 1, "prefill": 0, "q_max": 1, "kv_max": 100000, "spread": 0.0, "window": 1020, "sinks": 4},
        # 48 streams at 20000 to 200000 positions, 4 sinks and a window of 4096, 4 bits; pages between are given back
        {"name": "stream_48_q4", "kind": "attend", "cache": "q4_0", "heads": 32, "kv": 8, "hd": 128, "page": 64,
         "seqs": 48, "prefill": 0, "q_max": 1, "kv_max": 200000, "spread": 0.9, "window": 4096, "sinks": 4},
        # chunks of two long prompts by a window of 1500 and 70 sinks (a system prompt), heads of 256, f16
        {"name": "stream_chunks_f16", "kind": "attend", "cache": "f16", "heads": 16, "kv": 8, "hd": 256, "page": 32,
         "seqs": 2, "prefill": 2, "q_max": 1100, "kv_max": 9000, "spread": 0.4, "window": 1500, "sinks": 70},
        # one sequence's 4 drafted tokens without the draft's probabilities (looked up in the text)
        {"name": "verify_1x4", "kind": "verify", "seqs": 1, "drafts": 4, "vocab": 151936, "by_logits": False,
         "top_k": 50, "top_p": 0.95, "min_p": 0.0, "greedy": 0.0, "std": 2.5, "near": 0.9},
        # 40 sequences of up to 5 tokens of a draft model, nucleus sampling, a tenth of them greedy
        {"name": "verify_40x5", "kind": "verify", "seqs": 40, "drafts": 5, "vocab": 128256, "by_logits": True,
         "top_k": 0, "top_p": 0.9, "min_p": 0.0, "greedy": 0.1, "std": 2.5, "near": 0.7},
        # one token with one adapter of rank 16
        {"name": "lora_1", "kind": "lora", "type": "f16", "tokens": 1, "k": 4096, "rows": 4096, "rank": 16,
         "adapters": 8, "shape": "decode", "without": 0.0, "ragged": False},
        # 64 requests' next tokens, 40 adapters, ranks up to 32, a tenth of the requests without one
        {"name": "lora_64", "kind": "lora", "type": "bf16", "tokens": 64, "k": 4096, "rows": 6144, "rank": 32,
         "adapters": 40, "shape": "decode", "without": 0.1, "ragged": True},
        # prompts of 7 requests, 5000 tokens together, to the rows of a gate projection
        {"name": "lora_prompts", "kind": "lora", "type": "bf16", "tokens": 5000, "k": 4096, "rows": 12288, "rank": 64,
         "adapters": 7, "shape": "prompts", "without": 0.0, "ragged": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "verify", "verify", "lora", "lora"])
    if kind == "lora":
        shape = rng.choice(["decode", "decode", "prompts"])
        c = {"kind": kind, "type": rng.choice(["f16", "bf16", "bf16", "f32"]),
             "tokens": _log(rng, 1, 300) if shape == "decode" else _log(rng, 20, 5000), "k": 32 * _log(rng, 4, 384),
             "rows": _log(rng, 60, 14000), "rank": 8 * rng.choice([1, 1, 2, 2, 3, 4, 8, 16]),
             "adapters": _log(rng, 1, 60), "shape": shape, "without": rng.choice([0.0, 0.1, 0.5]),
             "ragged": rng.random() < 0.5}
        # at most what lora_prompts moves and multiplies, and the adapters within 1 GB
        while c["tokens"] * (c["k"] + 2 * c["rows"]) > 5000 * (4096 + 2 * 12288) or \
                c["tokens"] * c["rank"] * (c["k"] + c["rows"]) > 5000 * 64 * (4096 + 12288):
            c["tokens"] = c["tokens"] * 2 // 3
        return c
    if kind == "verify":
        vocab = _log(rng, 1000, 262144)
        drafts = rng.choice([0, 1, 2, 3, 4, 5, 8])
        return {"kind": kind, "drafts": drafts, "vocab": vocab,
                "seqs": max(1, min(_log(rng, 1, 64), 40 * 6 * 128256 // (vocab * (drafts + 1)))),
                "by_logits": rng.random() < 0.6, "top_k": rng.choice([0, 0, 1, 50, _log(rng, 2, 2000)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.05, 0.999), 3)]),
                "min_p": rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]), "greedy": rng.choice([0.0, 0.2]),
                "std": round(rng.uniform(0.3, 4.0), 2), "near": round(rng.uniform(0.0, 1.0), 2)}
    kv = rng.choice([1, 2, 4, 8])
    hd = rng.choice([64, 128, 128, 256])
    c = {"kind": kind, "heads": kv * rng.choice([1, 2, 3, 4, 5, 8]), "kv": kv, "hd": hd,
         "page": rng.choice([16, 32, 64, 128, 256])}
    shape = rng.choice(["decode", "decode", "few", "prompt", "mixed"])
    if kind == "append":
        seqs = _log(rng, 1, 256) if shape in ("decode", "few") else rng.randint(1, 8)
        q_max = {"decode": 1, "few": rng.randint(2, 8)}.get(shape) or _log(rng, 33, 4096)
        q_max = max(1, min(q_max, 8192 * 48 * 128 // ((c["heads"] + 2 * kv) * hd * seqs)))
        c.update(seqs=seqs, prefill=0 if shape == "decode" else 1 if shape == "mixed" else seqs, q_max=q_max,
                 kv_max=max(q_max, _log(rng, 1, 200000)), spread=round(rng.uniform(0, 0.95), 2),
                 norm=rng.random() < 0.7, base=rng.choice([1e4, 5e5, 1e6]))
        return c
    cache = rng.choice(["e4m3", "e4m3", "f16", "q4_0"])
    window, sinks = (0, 0) if cache == "e4m3" and rng.random() < 0.5 else (_log(rng, 16, 4096), _log(rng, 1, 300))
    seqs = _log(rng, 1, 64) if shape in ("decode", "few") else rng.randint(1, 12)
    q_max = {"decode": 1, "few": rng.randint(2, 8)}.get(shape) or _log(rng, 33, 2048)
    kv_max = max(q_max, _log(rng, 1, 200000 if window else 32000))
    if not window:  # no more positions than the 64 sequences of 820 to 8192 with 8 kv heads of 128
        kv_max = max(q_max, min(kv_max, 35 * 8192 * 8 * 128 // (seqs * kv * hd)))
    n_pre = 0 if shape == "decode" else 1 if shape == "mixed" else seqs
    seen = lambda: min(kv_max, window + sinks + q_max) if window else kv_max  # noqa: E731
    # the flops of the longest chunk; the plain form pads every sequence to the longest, its scores within 8 GB
    while n_pre and n_pre * q_max * seen() * c["heads"] * hd > 2048 * 8000 * 32 * 128:
        q_max = max(1, q_max // 2)
        kv_max = max(q_max, kv_max * 2 // 3)
    while seqs > 1 and seqs * q_max * seen() * c["heads"] > 2_000_000_000:
        seqs = max(1, seqs // 2)
        n_pre = min(n_pre, seqs)
    c.update(cache=cache, seqs=seqs, prefill=n_pre, q_max=q_max, kv_max=kv_max, spread=round(rng.uniform(0, 0.95), 2),
             window=window, sinks=sinks)
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


def _hidden(c, n, end):
    """The positions [a, b) of a sequence of `end` positions that none of its last n sees."""
    b = max(0, end - n + 1 - c["window"]) if c["window"] else 0
    return min(c["sinks"], b), b


def _row_bytes(c):
    return {"f16": c["hd"] * 2, "q4_0": c["hd"] // 2 + c["hd"] // 16, "e4m3": c["hd"]}[c.get("cache", "e4m3")]


def _head_bytes(c):
    """Of one head's K or V in a page."""
    return c["page"] * _row_bytes(c) + (16 if c.get("cache", "e4m3") == "e4m3" else 0)


def _draft_rows(c):
    """Rows of logits of every sequence: one more than it has drafted tokens."""
    return [1 + max(0, c["drafts"] - (i * 3) % 4 // 2) for i in range(c["seqs"])]


def _adapters(c):
    """The adapter of every token, -1 where it has none: one a request."""
    n = c["adapters"]
    pick = lambda i: -1 if (i * 0.7548776662 + 0.3) % 1 < c["without"] else int(i * 0.6180339887 % 1 * n)  # noqa: E731
    if c["shape"] == "decode":
        return [pick(i) for i in range(c["tokens"])]
    # a prompt for every adapter, longer and shorter ones
    part = [1 + (i * 0.7548776662) % 1 for i in range(n)]
    ends = [round(c["tokens"] * sum(part[:i + 1]) / sum(part)) for i in range(n)]
    got, i = [], 0
    for t in range(c["tokens"]):
        while t >= ends[i]:
            i += 1
        got.append(-1 if (i * 0.7548776662 + 0.3) % 1 < c["without"] else i)
    return got


def _ranks(c):
    return [max(1, c["rank"] - i * 5 % c["rank"]) if c["ragged"] else c["rank"] for i in range(c["adapters"])]


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


def _starts(q):
    at = [0]
    for n in q:
        at.append(at[-1] + n)
    return at


def _pages(c, g):
    """(table of pages, pages): every sequence's pages scattered over the pool.  -1 stands where a sequence has no
    page: an append's table names the pages that it writes only, an attention's none that lies wholly between the
    sinks and what its window reaches."""
    q, kv = _lens(c)
    page = c["page"]
    spans = []
    for n, end in zip(q, kv):
        last = (end + page - 1) // page
        if c["kind"] == "append":
            spans.append([((end - n) // page, last)])
        else:
            a, b = _hidden(c, n, end)
            cut = (a + page - 1) // page
            spans.append([(0, last)] if b // page <= cut else [(0, cut), (b // page, last)])
    total = sum(b - a for s in spans for a, b in s)
    order = g.order(total).to(torch.int32).cpu()
    table = torch.full((c["seqs"], max(s[-1][1] for s in spans)), -1, dtype=torch.int32)
    at = 0
    for i, s in enumerate(spans):
        for a, b in s:
            table[i, a:b] = order[at:at + b - a]
            at += b - a
    return table.cuda(), total


def _cache_values(c, g, pages):
    """What a cache holds, by position, K then V: (values f16, None), (nibbles u8, scales f16 [.., hd/32]) or
    (e4m3 codes u8, scale bytes u8 [pages, kv, page/16]); each [pages, kv, page, hd]."""
    shape = (pages, c["kv"], c["page"], c["hd"])
    got = []
    for _ in range(2):
        x = g.normal(*shape)
        if c.get("cache", "e4m3") == "e4m3":
            # a block's largest lies between 224 and 448 of its scale; the scales of what heads hold differ
            k = (g.uniform(*shape[:2], c["page"] // 16) * 4).floor_() - 9
            codes = (x * 80).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            got.append((codes, (k + 127).to(torch.uint8)))
        elif c["cache"] == "f16":
            got.append((x.half(), None))
        else:
            n = (x * 2.8 + 8.5).floor_().clamp_(0, 15).to(torch.uint8)
            d = (0.3 * (1 + 0.1 * g.normal(*shape[:3], shape[3] // 32))).bfloat16().half()
            got.append((n, d))
    return got


def _with_scales(c, codes, scales):
    """Codes [pages, kv, page * hd] and the 16 bytes of their scales behind."""
    pad = torch.zeros(*scales.shape[:2], 16 - scales.shape[2], dtype=torch.uint8, device="cuda")
    return torch.cat([codes, scales, pad], 2)


def _pack_k(c, v, d):
    """K's pool, bytes [pages, kv, head bytes]."""
    p = v.shape[0]
    if d is None:
        return v.reshape(p, c["kv"], -1).view(torch.uint8).clone()
    if d.dtype == torch.uint8:
        return _with_scales(c, v.reshape(p, c["kv"], -1), d)
    b = v.reshape(p, c["kv"], c["page"], c["hd"] // 32, 2, 16)
    nib = (b[..., 0, :] | (b[..., 1, :] << 4)).reshape(p, c["kv"], -1)
    return torch.cat([nib, d.reshape(p, c["kv"], -1).view(torch.uint8)], 2)


def _pack_v(c, v, d):
    """V's pool, bytes [pages, kv, head bytes]."""
    p, groups = v.shape[0], c["page"] // 8
    if d is None or d.dtype == torch.uint8:
        x = v.reshape(p, c["kv"], groups, 8, c["hd"]).transpose(3, 4).reshape(p, c["kv"], -1)
        return x.view(torch.uint8) if d is None else _with_scales(c, x, d)
    b = v.reshape(p, c["kv"], groups, 4, 2, c["hd"])  # positions 2i and 2i + 1
    halves = [sum(b[..., i, h, :].to(torch.int32) << (4 * i) for i in range(4)) for h in range(2)]
    words = (halves[0] | (halves[1] << 16)).reshape(p, c["kv"], -1)
    s = d.reshape(p, c["kv"], groups, 8, c["hd"] // 32).transpose(3, 4).reshape(p, c["kv"], -1)
    return torch.cat([words.view(torch.uint8), s.view(torch.uint8)], 2)


class _State:
    pass


def _logits(c, g):
    """(target, draft) rows as two models of one text give them: alike up to a share, a few tokens stand out."""
    rows = sum(_draft_rows(c))
    lead = (torch.arange(8, device="cuda") * 0.6180339887 * c["vocab"]).long() % c["vocab"]
    x = c["std"] * g.normal(rows, c["vocab"])
    x[:, lead] += 2.0 * c["std"]
    y = math.sqrt(1 - c["near"] ** 2) * c["std"] * g.normal(rows, c["vocab"])
    return x, y.add_(x, alpha=c["near"])


def _verify_inputs(c, g):
    """target, draft, drafted tokens, temperatures, numbers for the acceptance and for the draws."""
    x, y = _logits(c, g)
    rows = x.shape[0]
    t = 0.5 + g.uniform(rows)
    t[g.uniform(rows) < c["greedy"]] = 0.0
    # drawn from the draft with the same filters, or looked up: what is likeliest elsewhere
    if c["by_logits"]:
        run_up = _probabilities(y, t, *_filters(c, rows)).cumsum(1)
        token = (run_up <= g.uniform(rows).double()[:, None] * run_up[:, -1:]).sum(1)
    else:
        token = y.argmax(1)
    return x, y, token.to(torch.int32), t, g.uniform(rows), g.uniform(c["seqs"])


def _filters(c, rows):
    full = lambda v, kind: torch.full((rows,), v, dtype=kind, device="cuda")  # noqa: E731
    return full(c["top_k"], torch.int32), full(c["top_p"], torch.float32), full(c["min_p"], torch.float32)


def _lora_inputs(c, g):
    kind = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[c["type"]]
    a = (g.normal(c["adapters"], c["rank"], c["k"]) * c["k"] ** -0.5).to(kind)
    b = (g.normal(c["adapters"], c["rows"], c["rank"]) * 0.2).to(kind)
    scale = 0.5 + g.uniform(c["adapters"])
    return a, b, scale, g.normal(c["tokens"], c["k"]), g.normal(c["tokens"], c["rows"])


def _append_inputs(c, g):
    q, kv = _lens(c)
    table, pages = _pages(c, g)
    qkv = g.normal(sum(q), (c["heads"] + 2 * c["kv"]) * c["hd"])
    qn, kn = 1 + 0.1 * g.normal(c["hd"]), 1 + 0.1 * g.normal(c["hd"])
    return q, kv, table, pages, qkv, qn, kn, _cache_values(c, g, pages)


def _attend_inputs(c, g):
    q, kv = _lens(c)
    table, pages = _pages(c, g)
    x = 1.5 * g.normal(sum(q), c["heads"], c["hd"])
    return q, kv, table, pages, x, _cache_values(c, g, pages)


def prepare(case, seed):
    c, g, s = case, _Inputs(seed), _State()
    s.case = c
    if c["kind"] == "lora":
        s.a, s.b, s.scale, s.x, s.res = _lora_inputs(c, g)
        s.adapter, s.ranks = _ints(_adapters(c)), _ints(_ranks(c))
        s.y = torch.empty_like(s.res)
    elif c["kind"] == "verify":
        s.target, s.draft, s.token, s.temperature, s.u, s.u_draw = _verify_inputs(c, g)
        s.rows = s.target.shape[0]
        s.top_k, s.top_p, s.min_p = _filters(c, s.rows)
        s.q_start = _ints(_starts(_draft_rows(c)))
        s.accepted = torch.empty(c["seqs"], dtype=torch.int32, device="cuda")
        s.out = torch.empty(s.rows, dtype=torch.int32, device="cuda")
    else:
        if c["kind"] == "append":
            q, kv, s.table, s.pages, s.qkv, s.qn, s.kn, (k, v) = _append_inputs(c, g)
            # the batch's rows and those before them in a block that they find begun
            s.back = [n + (end - n) % 16 for n, end in zip(q, kv)]
            s.back_start, s.back_tokens = _ints(_starts(s.back)), sum(s.back)
            s.q_out = torch.empty(sum(q), c["heads"], c["hd"], device="cuda")
            s.k_out, s.v_out = (torch.empty(s.back_tokens, c["kv"], c["hd"], device="cuda") for _ in range(2))
        else:
            q, kv, s.table, s.pages, s.q, (k, v) = _attend_inputs(c, g)
            s.out = torch.empty_like(s.q)
            s.most = max(end - b + a for n, end in zip(q, kv) for a, b in [_hidden(c, n, end)])
        s.k_pool, s.v_pool = _pack_k(c, *k), _pack_v(c, *v)
        s.tokens, s.longest = sum(q), max(q)
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
    ptr = lambda t: t.data_ptr()  # noqa: E731
    if c["kind"] == "lora":
        kind = {"f16": zd.F16, "bf16": zd.BF16, "f32": zd.F32}[c["type"]]
        lora = zd.Lora(ptr(s.a), ptr(s.b), kind, c["adapters"], c["rank"], c["rows"], c["k"],
                       ranks=ptr(s.ranks) if c["ragged"] else 0, scales=ptr(s.scale))
        if not d.lora_enqueue(lora, c["tokens"], ptr(s.adapter), ptr(s.x), ptr(s.y), res=ptr(s.res)):
            raise RuntimeError(d.last_error())
        return s.y
    if c["kind"] == "verify":
        how = zd.Sampling(temperature=ptr(s.temperature), top_k=ptr(s.top_k), top_p=ptr(s.top_p), min_p=ptr(s.min_p))
        draft = {"draft_logits": ptr(s.draft), "draft_how": how} if c["by_logits"] else {}
        if not d.verify_enqueue(ptr(s.target), s.rows, c["vocab"], c["seqs"], ptr(s.q_start), ptr(s.token), ptr(s.u),
                                ptr(s.u_draw), ptr(s.accepted), ptr(s.out), how=how, **draft):
            raise RuntimeError(d.last_error())
        return {"accepted": s.accepted, "token": s.out}
    kind = {"f16": zd.F16, "q4_0": zd.Q4_0, "e4m3": zd.CACHE_E4M3}[c.get("cache", "e4m3")]
    cache = zd.PagedCache(ptr(s.k_pool), ptr(s.v_pool), kind, c["kv"], c["hd"], c["page"], s.pages)
    batch = zd.PagedBatch(c["seqs"], s.tokens, ptr(s.q_start), ptr(s.kv_len), ptr(s.table), s.table.shape[1])
    if c["kind"] == "attend":
        if not d.paged_attention_enqueue(cache, batch, ptr(s.q), ptr(s.out), c["heads"], c["hd"] ** -0.5,
                                         window=c["window"], sinks=c["sinks"]):
            raise RuntimeError(d.last_error())
        return s.out
    norm = (ptr(s.qn), ptr(s.kn)) if c["norm"] else (0, 0)
    back = zd.PagedBatch(c["seqs"], s.back_tokens, ptr(s.back_start), ptr(s.kv_len), ptr(s.table), s.table.shape[1])
    if not (d.paged_append_enqueue(cache, batch, ptr(s.qkv), ptr(s.q_out), c["heads"], EPS, c["base"],
                                   q_norm_w=norm[0], k_norm_w=norm[1]) and
            d.paged_read_enqueue(cache, back, ptr(s.k_out), ptr(s.v_out))):
        raise RuntimeError(d.last_error())
    return {"q": s.q_out, "k": s.k_out, "v": s.v_out}


# ---- one pass: the plain form -------------------------------------------------------------


def _token_places(q_start, kv_len, tokens):
    """(sequence, position) of every token of a batch."""
    t = torch.arange(tokens, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(q_start[1:].contiguous(), t, right=True)
    pos = kv_len[seq] - (q_start[seq + 1] - q_start[seq]) + (t - q_start[seq])
    return seq, pos.long()


def _rotated(c, x, w, pos):
    """x (float64, [tokens, heads, hd]): head norm, then the rotation by the position."""
    if c["norm"]:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    half = c["hd"] // 2
    inv = torch.pow(torch.tensor(c["base"], dtype=torch.float64, device="cuda"),
                    torch.arange(half, dtype=torch.float64, device="cuda") * (-2.0 / c["hd"]))
    a = (pos.double()[:, None] * inv)[:, None, :]
    cos, sin = a.cos(), a.sin()
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], -1)


def _two(k):
    """2^k, exactly (float64)."""
    return ((k.long() + 1023) << 52).view(torch.float64)


def _e4m3(x, k):
    """The e4m3 numbers nearest to x / 2^k (float64; k broadcasts)."""
    y = x * _two(-k)
    step = _two(torch.frexp(y)[1].clamp_min(-5) - 4)  # 2^(e - 3) for 2^e <= |y|, e >= -6
    return (torch.round(y / step) * step).clamp(-448, 448)


def _codes(y):
    return y.float().to(torch.float8_e4m3fn).view(torch.uint8)


def _numbers(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _places_of(c, s, seq, pos):
    """The places of positions in the pools' views: page, block of 16, offset."""
    return s.table[seq, pos // c["page"]].long(), (pos % c["page"]) // 16, pos % c["page"]


def _pool_views(c, s):
    """Codes of K [pages, kv, page, hd] and of V [pages, kv, page/8, hd, 8], scale bytes [pages, kv, page/16]."""
    n = c["page"] * c["hd"]
    k = s.k_pool[:, :, :n].unflatten(2, (c["page"], c["hd"]))
    v = s.v_pool[:, :, :n].unflatten(2, (c["page"] // 8, c["hd"], 8))
    scales = [t[:, :, n:n + c["page"] // 16] for t in (s.k_pool, s.v_pool)]
    return (k, scales[0]), (v, scales[1])


def _append_plain(s):
    c = s.case
    kv, hd = c["kv"], c["hd"]
    seq, pos = _token_places(s.q_start, s.kv_len, s.tokens)
    x = s.qkv.double().reshape(s.tokens, -1, hd)
    q = _rotated(c, x[:, :c["heads"]], s.qn, pos).float()
    new = _rotated(c, x[:, c["heads"]:c["heads"] + kv], s.kn, pos), x[:, c["heads"] + kv:]
    p, blk, off = _places_of(c, s, seq, pos)
    heads = torch.arange(kv, device="cuda")
    # rows before the batch's in blocks that it finds begun
    back_seq, back_pos = _token_places(s.back_start, s.kv_len, s.back_tokens)
    old = back_pos < (s.kv_len - (s.q_start[1:] - s.q_start[:-1]))[back_seq]
    o_seq, o_pos = back_seq[old], back_pos[old]
    op, oblk, ooff = _places_of(c, s, o_seq, o_pos)
    out = {"q": q}
    for name, values, (codes, scales) in zip("kv", new, _pool_views(c, s)):
        # the scale that the largest of a block's new values needs, no smaller than one that it has
        need = torch.full((s.pages, c["page"] // 16, kv), K_MIN, dtype=torch.int64, device="cuda")
        m, e = torch.frexp(values.abs().amax(-1) / 448)
        e = torch.where(m > 0.5, e, e - 1).clamp(K_MIN, K_MAX).long()
        flat = need.view(-1, kv)
        at = (p * (c["page"] // 16) + blk)[:, None].expand(-1, kv)
        flat.scatter_reduce_(0, at, e, "amax")
        had = scales[op, :, oblk].long() - 127
        flat.scatter_reduce_(0, (op * (c["page"] // 16) + oblk)[:, None].expand(-1, kv), had, "amax")
        if name == "k":
            view = lambda pg, o: (pg[:, None], heads[None], o[:, None])  # noqa: E731
        else:
            view = lambda pg, o: (pg[:, None], heads[None], o[:, None] // 8, slice(None), o[:, None] % 8)  # noqa: E731
        # what was there at the new scale, then the new rows
        was = _numbers(codes[view(op, ooff)]).double()
        kept = _codes(_e4m3(was * _two(had)[..., None], need[op, oblk][..., None]))
        codes[view(op, ooff)] = kept
        codes[view(p, off)] = _codes(_e4m3(values, need[p, blk][..., None]))
        scales[op, :, oblk] = (need[op, oblk] + 127).to(torch.uint8)
        scales[p, :, blk] = (need[p, blk] + 127).to(torch.uint8)
        bp, bblk, boff = _places_of(c, s, back_seq, back_pos)
        k = scales[bp, :, bblk].long() - 127
        out[name] = _numbers(codes[view(bp, boff)]) * _two(k).float()[..., None]
    return out


def _rows_at(c, s, seq, pos):
    """K and V float32 [.., kv, hd] of positions [..] of sequences [..] (0 where there is no page)."""
    hd, page = c["hd"], c["page"]
    p = s.table[seq, pos // page].long()
    none = (p < 0)[..., None, None]
    p, off = p.clamp_min(0), pos % page
    g, j = off // 8, off % 8
    nib = page * hd // 2
    if c["cache"] == "f16":
        k = s.k_pool.view(torch.float16).unflatten(2, (page, hd))[p, :, off].float()
        v = s.v_pool.view(torch.float16).unflatten(2, (page // 8, hd, 8))[p, :, g, :, j].float()
    elif c["cache"] == "e4m3":
        (kc, ks), (vc, vs) = _pool_views(c, s)
        k = _numbers(kc[p, :, off]) * _two(ks[p, :, off // 16].long() - 127).float()[..., None]
        v = _numbers(vc[p, :, g, :, j]) * _two(vs[p, :, off // 16].long() - 127).float()[..., None]
    else:
        b = s.k_pool[:, :, :nib].unflatten(2, (page, hd // 32, 16))[p, :, off]
        d = s.k_pool[:, :, nib:].view(torch.float16).unflatten(2, (page, hd // 32))[p, :, off].float()
        k = ((torch.cat([b & 15, b >> 4], -1).float() - 8) * d[..., None]).flatten(-2)
        w = s.v_pool[:, :, :nib].view(torch.int32).unflatten(2, (page // 8, hd))[p, :, g]
        w = (w >> (4 * (j // 2) + 16 * (j % 2)).int()[..., None, None]) & 15
        d = s.v_pool[:, :, nib:].view(torch.float16).unflatten(2, (page // 8, hd // 32, 8))[p, :, g, :, j].float()
        v = ((w.unflatten(-1, (-1, 32)).float() - 8) * d[..., None]).flatten(-2)
    return k.masked_fill_(none, 0), v.masked_fill_(none, 0)


def _attend_plain(s):
    c = s.case
    kv, hd, g, n = c["kv"], c["hd"], c["heads"] // c["kv"], c["seqs"]
    seq, pos = _token_places(s.q_start, s.kv_len, s.tokens)
    # the positions that any row of a sequence sees, its sinks and then the others, as far as the most of them
    lens = s.q_start[1:] - s.q_start[:-1]
    first = (s.kv_len - lens + 1 - c["window"]).clamp_min(0)[:, None] if c["window"] else torch.zeros_like(lens)[:, None]
    j = torch.arange(s.most, device="cuda")[None].expand(n, -1)
    at_sink = torch.clamp(first, max=c["sinks"])
    at = torch.where(j < at_sink, j, j + (first - at_sink)).long()
    inside = at < s.kv_len[:, None]
    k, v = _rows_at(c, s, torch.arange(n, device="cuda")[:, None].expand_as(at), torch.where(inside, at, 0))
    k, v = (x.permute(0, 2, 1, 3).reshape(n * kv, -1, hd) for x in (k, v))
    row = torch.arange(s.tokens, device="cuda") - s.q_start[seq]
    q = torch.zeros(n, s.longest, kv, g, hd, device="cuda")
    q[seq, row] = s.q.view(s.tokens, kv, g, hd)
    q = q.permute(0, 2, 1, 3, 4).reshape(n * kv, s.longest * g, hd)
    of = torch.full((n, s.longest), -1, dtype=torch.long, device="cuda")
    of[seq, row] = pos
    seen = (at[:, None] <= of[..., None]) & inside[:, None]
    if c["window"]:
        seen &= (at[:, None] > of[..., None] - c["window"]) | (at[:, None] < c["sinks"])
    scores = torch.bmm(q * hd ** -0.5, k.transpose(1, 2).contiguous())
    scores = scores.view(n, kv, s.longest, g, -1).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.bmm(scores.view(n * kv, s.longest * g, -1), v)
    out = out.view(n, kv, s.longest, g, hd) / total
    return out.permute(0, 2, 1, 3, 4)[seq, row].reshape(s.tokens, c["heads"], hd)


def _probabilities(logits, temperature, top_k, top_p, min_p):
    """What a draw with these filters takes a row's tokens by (float64)."""
    x, at = torch.sort(logits, dim=1, descending=True, stable=True)
    rank = torch.arange(x.shape[1], device="cuda")
    t = temperature.double()[:, None]
    x = x.double()
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    k = top_k.long()[:, None]
    w = torch.where((k <= 0) | (rank < k), w, 0.0)
    run_up = w.cumsum(1)
    w = torch.where(run_up - w < top_p.double()[:, None] * run_up[:, -1:], w, 0.0)
    w = torch.where(w >= min_p.double()[:, None], w, 0.0)
    w = torch.where((t > 0) | (rank < 1), w, 0.0)  # temperature 0: the largest
    return torch.zeros_like(w).scatter_(1, at, w / w.sum(1, keepdim=True))


def _verify_plain(s):
    c = s.case
    n, rows = c["seqs"], s.rows
    how = (s.temperature, s.top_k, s.top_p, s.min_p)
    p = _probabilities(s.target, *how)
    d = s.token.long()[:, None]
    if c["by_logits"]:
        q = _probabilities(s.draft, *how)
    else:
        q = torch.zeros_like(p).scatter_(1, d, 1.0)
    r = torch.arange(rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s.q_start[1:].contiguous(), r, right=True)
    last = r + 1 == s.q_start[seq + 1]
    yes = (s.u.double() * torch.gather(q, 1, d)[:, 0] < torch.gather(p, 1, d)[:, 0]) & ~last
    # the first row of a sequence that is not accepted
    stop = torch.full((n,), rows, dtype=torch.int64, device="cuda")
    stop.scatter_reduce_(0, seq, torch.where(yes, rows, r.long()), "amin")
    w = torch.where(last[stop][:, None], p[stop], (p[stop] - q[stop]).clamp_min(0))
    w = torch.where(w.sum(1, keepdim=True) > 0, w, p[stop])
    run_up = w.cumsum(1)
    drawn = (run_up <= s.u_draw.double()[:, None] * run_up[:, -1:]).sum(1)
    token = torch.where(r < stop[seq], s.token, torch.where(r == stop[seq], drawn[seq].int(), -1))
    return {"accepted": (stop - s.q_start[:-1]).int(), "token": token.int()}


def _lora_plain(s):
    c = s.case
    y = s.res.clone()
    live = torch.arange(c["rank"], device="cuda")[None] < s.ranks[:, None]
    for i in range(c["adapters"]):
        at = torch.nonzero(s.adapter == i)[:, 0]
        if not len(at):
            continue
        h = s.x[at] @ s.a[i].float().T
        y[at] += s.scale[i] * ((h * live[i]) @ s.b[i].float().T)
    return y


def run(state):
    if own:
        return _run_own(state)
    return {"append": _append_plain, "attend": _attend_plain, "verify": _verify_plain,
            "lora": _lora_plain}[state.case["kind"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    c = case
    if c["kind"] == "lora":
        used, ranks = [i for i in _adapters(c) if i >= 0], _ranks(c)
        size = 4 if c["type"] == "f32" else 2
        return {"bytes": 4 * len(used) * c["k"] + 8 * c["tokens"] * c["rows"] + 4 * c["tokens"]
                + size * (c["k"] + c["rows"]) * sum(ranks[i] for i in set(used)),
                "flops": 2 * (c["k"] + c["rows"]) * sum(ranks[i] for i in used)}
    if c["kind"] == "verify":
        rows = _draft_rows(c)
        read = sum(rows) + (sum(n - 1 for n in rows) if c["by_logits"] else 0)
        return {"bytes": 4 * read * c["vocab"] + 28 * sum(rows) + 8 * c["seqs"], "flops": 8 * read * c["vocab"]}
    q, kv = _lens(c)
    tokens, head = sum(q), c["kv"] * c["hd"]
    if c["kind"] == "append":
        back = sum(n + (end - n) % 16 for n, end in zip(q, kv))
        return {"bytes": tokens * (8 * c["heads"] * c["hd"] + 8 * head + 2 * head) + 8 * back * head,
                "flops": tokens * 12 * (c["heads"] + 2 * c["kv"]) * c["hd"]}
    cached = pairs = pages = 0
    for n, end in zip(q, kv):
        a, b = _hidden(c, n, end)
        cached += end - b + a
        pages += (end - b + a + c["page"] - 1) // c["page"]
        w = c["window"] or end
        pairs += sum(min(p + 1, w) + min(c["sinks"], max(0, p + 1 - w)) for p in range(end - n, end))
    return {"bytes": 2 * cached * c["kv"] * _row_bytes(c) + 8 * tokens * c["heads"] * c["hd"] + 4 * pages,
            "flops": 4 * pairs * c["heads"] * c["hd"]}


# ---- the same in 64 bits, from the definitions ------------------------------------------------


def _rope64(x, base, pos):
    """x [n, heads, hd] float64 as complex pairs (i, i + hd/2) turned by pos * base^(-2i/hd)."""
    n = x.shape[-1] // 2
    i = torch.arange(n, dtype=torch.float64, device=x.device)
    turn = torch.exp(i * (-2.0 / x.shape[-1]) * math.log(base))[None, :] * pos[:, None]
    z = torch.complex(x[..., :n], x[..., n:]) * torch.polar(torch.ones_like(turn), turn)[:, None, :]
    return torch.cat([z.real, z.imag], -1)


def _e4m3_set():
    """The e4m3 numbers of 0 and above in order of their codes 0 to 126, by the format's definition."""
    got = []
    for b in range(127):
        e, m = b >> 3, b & 7
        got.append(math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10))
    return torch.tensor(got, dtype=torch.float64, device="cuda")


def _nearest(x, numbers):
    """The numbers nearest to x, of two equally near the one whose code is even."""
    a = x.abs().contiguous()
    hi = torch.searchsorted(numbers, a).clamp(1, 126)
    lo = hi - 1
    below, above = a - numbers[lo], numbers[hi] - a
    pick = torch.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, lo)
    return torch.copysign(numbers[pick], x)


def _append_exact(c, g):
    q, kv, table, pages, qkv, qn, kn, cache = _append_inputs(c, g)
    x = qkv.double().reshape(sum(q), -1, c["hd"])
    pos = torch.cat([torch.arange(end - n, end, dtype=torch.float64, device="cuda") for n, end in zip(q, kv)])

    def head(y, w):
        if c["norm"]:
            y = y * torch.rsqrt(y.pow(2).sum(-1, keepdim=True) / c["hd"] + EPS) * w.double()
        return _rope64(y, c["base"], pos)

    h, page, numbers = c["heads"], c["page"], _e4m3_set()
    new = {"k": head(x[:, h:h + c["kv"]], kn), "v": x[:, h + c["kv"]:]}
    got = {"q": head(x[:, :h], qn), "k": [], "v": []}
    table, at = table.cpu(), 0
    limits = torch.tensor([448 * 2.0 ** k for k in range(K_MIN, K_MAX)], dtype=torch.float64, device="cuda")
    units = torch.tensor([2.0 ** k for k in range(K_MIN, K_MAX + 1)], dtype=torch.float64, device="cuda")
    for i, (n, end) in enumerate(zip(q, kv)):
        first = end - n
        for name, (codes, scales) in zip("kv", cache):
            rows = new[name][at:at + n]
            begun = first % 16
            # the begun block's rows, and all rows filled up to whole blocks with zeros
            page_id, off = int(table[i, first // page]), first % page // 16
            old = codes[page_id, :, off * 16:off * 16 + begun].transpose(0, 1)
            k0 = scales[page_id, :, off].long() - 127 - K_MIN
            b = old.long() & 127
            was = torch.where(old >= 128, -1.0, 1.0) * numbers[b] * units[k0][None, :, None]
            fill = rows.new_zeros((-end) % 16, *rows.shape[1:])
            blocks = torch.cat([rows.new_zeros(begun, *rows.shape[1:]), rows, fill]).unflatten(0, (-1, 16))
            top = blocks.abs().amax((1, 3))  # [blocks, kv]
            k = (top[..., None] > limits).sum(-1)  # over K_MIN
            if begun:
                k[0] = torch.maximum(k[0], k0)
                blocks[0, :begun] = was
            unit = units[k][:, None, :, None]
            held = (_nearest(blocks / unit, numbers) * unit).flatten(0, 1)
            got[name].append(held[:begun + n])
        at += n
    return {"q": got["q"], "k": torch.cat(got["k"]), "v": torch.cat(got["v"])}


def _attend_exact(c, g):
    q, kv, table, _, x, (k, v) = _attend_inputs(c, g)
    table = table.long()
    out, at, group = [], 0, c["heads"] // c["kv"]
    numbers = torch.cat([_e4m3_set(), torch.tensor([math.nan], dtype=torch.float64, device="cuda")])
    units = torch.tensor([2.0 ** k for k in range(K_MIN, K_MAX + 1)], dtype=torch.float64, device="cuda")

    def rows(values, scales, pages):
        y = values[pages]
        if scales is None:
            y = y.double()
        elif scales.dtype == torch.uint8:
            s = units[scales[pages].long() - 127 - K_MIN]
            y = numbers[(y & 127).long()] * torch.where(y >= 128, -1.0, 1.0) * s.repeat_interleave(16, 2)[..., None]
        else:
            y = (y.double().unflatten(-1, (-1, 32)) - 8) * scales[pages].double().unsqueeze(-1)
            y = y.flatten(-2)
        return y.transpose(0, 1).flatten(1, 2)  # [kv, positions, hd]

    for i, (n, end) in enumerate(zip(q, kv)):
        ids = table[i, :(end + c["page"] - 1) // c["page"]]
        has = ids >= 0
        j = torch.arange(len(ids) * c["page"], device="cuda").view(-1, c["page"])[has].flatten()
        kk, vv = (rows(*t, ids[has]) for t in (k, v))
        p = torch.arange(end - n, end, device="cuda")[:, None]
        off = j[None] > p
        if c["window"]:
            off |= (j[None] <= p - c["window"]) & (j[None] >= c["sinks"])
        heads = []
        for h in range(c["heads"]):
            score = x[at:at + n, h].double() @ kk[h // group].T.contiguous() / math.sqrt(c["hd"])
            heads.append(torch.softmax(score.masked_fill(off, -math.inf), 1) @ vv[h // group])
        out.append(torch.stack(heads, 1))
        at += n
    return torch.cat(out)


def _kept(x, t, c):
    """The probabilities of a row (float64, by token) that is drawn from at temperature t with the case's filters."""
    p = torch.zeros_like(x)
    if t <= 0:
        p[int(x.argmax())] = 1.0
        return p
    order = torch.argsort(-x, stable=True)
    if c["top_k"] > 0:
        order = order[:c["top_k"]]
    v = torch.softmax(x[order] / t, 0)
    before = torch.cat([v.new_zeros(1), v.cumsum(0)[:-1]])
    single = lambda f: float(torch.tensor(f, dtype=torch.float32))  # noqa: E731
    keep = (before < single(c["top_p"])) & (v >= single(c["min_p"]) * v[0])
    p[order[keep]] = v[keep] / v[keep].sum()
    return p


def _verify_exact(c, g):
    x, y, token, t, u, u_draw = _verify_inputs(c, g)
    token, t, u, u_draw = token.tolist(), t.tolist(), u.tolist(), u_draw.tolist()
    accepted, out, row = [], [], 0
    for i, n in enumerate(_draft_rows(c)):
        got = []
        for j in range(n):
            r = row + j
            p, q = _kept(x[r].double(), t[r], c), None
            if j < n - 1:
                if c["by_logits"]:
                    q = _kept(y[r].double(), t[r], c)
                else:
                    q = torch.zeros_like(p)
                    q[token[r]] = 1.0
                if u[r] * float(q[token[r]]) < float(p[token[r]]):
                    got.append(token[r])
                    continue
                rest = (p - q).clamp_min(0)
                p = rest if float(rest.sum()) > 0 else p
            at = torch.searchsorted(p.cumsum(0), u_draw[i] * float(p.cumsum(0)[-1]), right=True)
            accepted.append(j)
            got.append(int(at))
            break
        out += got + [-1] * (n - len(got))
        row += n
    return {"accepted": torch.tensor(accepted, dtype=torch.int32), "token": torch.tensor(out, dtype=torch.int32)}


def _lora_exact(c, g):
    a, b, scale, x, res = _lora_inputs(c, g)
    y, ranks, of = res.double(), _ranks(c), torch.tensor(_adapters(c), device="cuda")
    for i in set(_adapters(c)) - {-1}:
        at = (of == i).nonzero()[:, 0]
        down, up = a[i, :ranks[i]].double(), b[i, :, :ranks[i]].double()
        y[at] += float(scale[i]) * (up @ (down @ x[at].double().T.contiguous())).T
    return y


def exact(case, seed):
    return {"append": _append_exact, "attend": _attend_exact, "verify": _verify_exact,
            "lora": _lora_exact}[case["kind"]](case, _Inputs(seed))
