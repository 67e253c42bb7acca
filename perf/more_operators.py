"""What the operators that a serving batch has per request are measured by: adapters beside shared projections, and a cache that is
kept to a budget by the attention its keys have received.

* ``weights``: the softmax weights that a step's query rows give to every cached key, added up per request and KV head, over pages
  in bfloat16 or in 8 bits (e4m3 codes, one power of two per row and plane).
* ``choose``: which places of every request and KV head are kept: the last ones, the first ones, then the largest sums (ties: the
  lowest place), in ascending order.
* ``compact``: the kept rows of keys and values, and their sums, moved to the front of other pages.
* ``adapt``: low-rank adapters of many requests beside a shared projection: out = y + scale_e (x A_e^T) B_e^T for every row's own e.

Plain forms are torch in 32 bits; ``exact`` restates them in 64, request by request."""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
FLOOR = 8192.0  # positions between two steps of the attention temperature


def _k():
    from jax_llm_examples_b200.kernels import api

    return api


# ------------------------------------------------------------------------------------------------------ the cases
def listed():
    plain = {"chunk": 0, "window": 0, "temper": 0.0, "cap": 0.0, "sink": False, "slopes": False}
    llama = {"heads": 40, "kv_heads": 8, "dim": 128, "page": 64}
    return [
        # one chat session: the latency of a token
        {"name": "weights_one", "kind": "weights", "cache": "bfloat16", "requests": 1, "tokens": 1, "context": 700, "ragged": False, **llama, **plain},
        # a serving batch of ragged sessions, a token each
        {"name": "weights_64", "kind": "weights", "cache": "bfloat16", "requests": 64, "tokens": 1, "context": 8192, "ragged": True, **llama, **plain},
        # a few long sessions over the 8-bit cache, with the temperature of far positions
        {"name": "weights_8_long_8bit", "kind": "weights", "cache": "float8", "requests": 8, "tokens": 1, "context": 30001, "ragged": True, **llama,
         **plain, "temper": 0.1},
        # prompts that just ended: the weights of their last 32 tokens decide what is kept of them
        {"name": "weights_last_32", "kind": "weights", "cache": "bfloat16", "requests": 8, "tokens": 32, "context": 8192, "ragged": True, **llama, **plain},
        # a whole prompt portion behind cached tokens, in the scheduler's default size
        {"name": "weights_portion_2048", "kind": "weights", "cache": "bfloat16", "requests": 1, "tokens": 2048, "context": 1500, "ragged": False, **llama,
         **plain},
        # one very long session is cut to its budget; a serving batch is
        {"name": "choose_one_long", "kind": "choose", "requests": 1, "kv_heads": 8, "length": 100001, "keep": 4096, "first": 4, "recent": 512, "ragged": False},
        {"name": "choose_64", "kind": "choose", "requests": 64, "kv_heads": 8, "length": 8192, "keep": 2048, "first": 4, "recent": 256, "ragged": True},
        # the kept rows of one session of small heads and pages in 8 bits; of a serving batch
        {"name": "compact_one_8bit", "kind": "compact", "cache": "float8", "requests": 1, "kv_heads": 4, "dim": 64, "page": 16, "length": 9001, "keep": 1500,
         "ragged": False},
        {"name": "compact_32", "kind": "compact", "cache": "bfloat16", "requests": 32, "kv_heads": 8, "dim": 128, "page": 64, "length": 8192, "keep": 2048,
         "ragged": True},
        # one session's token through its adapter beside the stacked q, k, v projection
        {"name": "adapt_one", "kind": "adapt", "dtype": "bfloat16", "out_dtype": "bfloat16", "rows": 1, "requests": 1, "adapters": 8, "rank": 16,
         "mixed_ranks": False, "k": 5120, "n": 7168, "bare": False},
        # a decode step of 64 sessions, some without an adapter, beside 32-bit partials of the same projection
        {"name": "adapt_64", "kind": "adapt", "dtype": "bfloat16", "out_dtype": "float32", "rows": 64, "requests": 64, "adapters": 24, "rank": 64,
         "mixed_ranks": True, "k": 5120, "n": 7168, "bare": True},
        # ragged prompt portions of three sessions
        {"name": "adapt_prompt_2048", "kind": "adapt", "dtype": "bfloat16", "out_dtype": "bfloat16", "rows": 2048, "requests": 3, "adapters": 8, "rank": 64,
         "mixed_ranks": False, "k": 5120, "n": 5120, "bare": False},
    ]


def _log(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# query heads, key/value heads, head size: this package's presets and their neighbours, groups of 1 to 16
HEADS = [(40, 8, 128), (32, 8, 128), (16, 4, 128), (16, 4, 64), (12, 12, 64), (16, 2, 128), (32, 2, 128), (6, 3, 64), (24, 8, 128), (8, 8, 128)]


def draw(rng):
    """Steps of serving batches of every size up to the listed ones."""
    kind = rng.choice(["weights", "weights", "choose", "compact", "adapt", "adapt"])
    if kind == "adapt":
        rows = _log(rng, 1, 2048)
        bits32 = rows <= 300 and rng.random() < 0.2
        rank = _log(rng, 1, 128) if rng.random() < 0.3 else rng.choice([8, 16, 16, 32, 64, 128])
        width = 1024 if bits32 else 5120
        sizes = [8 * _log(rng, 8, width // 8), 8 * _log(rng, 8, width // 8)]
        if rng.random() < 0.15:
            sizes = [sizes[0] + rng.randint(1, 7), sizes[1] + rng.randint(1, 7)]
        return {"kind": kind, "dtype": "float32" if bits32 else "bfloat16", "out_dtype": "float32" if bits32 else rng.choice(["bfloat16", "bfloat16", "float32"]),
                "rows": rows, "requests": min(rows, _log(rng, 1, 64)), "adapters": _log(rng, 1, 32), "rank": rank, "mixed_ranks": rng.random() < 0.4,
                "k": sizes[0], "n": sizes[1], "bare": rng.random() < 0.4}
    heads, kv_heads, dim = rng.choice(HEADS)
    ragged = rng.random() < 0.7
    if kind == "choose":
        length = _log(rng, 1, 131072)
        keep = _log(rng, 1, max(1, length)) if rng.random() < 0.9 else length + 5
        return {"kind": kind, "requests": _log(rng, 1, max(1, min(64, 500000 // length))), "kv_heads": kv_heads, "length": length, "keep": keep,
                "first": rng.choice([0, 1, 4]), "recent": rng.choice([0, _log(rng, 1, 512)]), "ragged": ragged}
    page = rng.choice([16, 32, 48, 64, 64, 64, 128])
    if kind == "compact":
        length = _log(rng, 2, 32768)
        return {"kind": kind, "cache": rng.choice(["bfloat16", "float8", "float32"]), "requests": _log(rng, 1, max(1, min(32, 100000 // length))),
                "kv_heads": kv_heads, "dim": dim, "page": page, "length": length, "keep": _log(rng, 1, length), "ragged": ragged}
    mask = rng.choice(["all", "all", "all", "chunk", "window"])
    case = {"kind": kind, "cache": rng.choice(["bfloat16", "bfloat16", "float8"]), "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "ragged": ragged,
            "chunk": _log(rng, 64, 8192) if mask == "chunk" else 0, "window": _log(rng, 16, 4096) if mask == "window" else 0,
            "temper": rng.choice([0.0, 0.0, 0.1]), "cap": rng.choice([0.0, 0.0, 0.0, 30.0]), "sink": rng.random() < 0.3, "slopes": rng.random() < 0.2}
    tokens = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 2048)])
    context = _log(rng, 1, 32768 if tokens == 1 else 8192 if tokens <= 64 else 3000)
    most = max(1, min(64, 390000 // context) if tokens == 1 else min(16, int(7e6 // (tokens * (context + tokens)))))
    return case | {"requests": _log(rng, 1, most), "tokens": tokens, "context": context}


# ----------------------------------------------------------------------------------------------------- the inputs
def _shares(case, least):
    """Lengths of the requests: the first in full, the others (ragged) down to half of it."""
    full = case["length"]
    return [max(least, full - (i * 2654435761 % 1000 * full // 2000 if case["ragged"] and i else 0)) for i in range(case["requests"])]


def _lengths(case):
    """(query rows of each request, keys it held before them): host lists."""
    R, T = case["requests"], case["tokens"]
    held = [max(0, case["context"] - (i * 2654435761 % 1000 * case["context"] // 2000 if case["ragged"] and i else 0)) for i in range(R)]
    n = [max(1, T - (i * 3 if case["ragged"] else 0)) for i in range(R)]
    return n, [c - 1 if m == 1 and c > 0 else c for c, m in zip(held, n)]


def _row_counts(case):
    """(Rows of each request, its adapter or -1): host lists."""
    N, R, E = case["rows"], case["requests"], case["adapters"]
    cuts = sorted({N * i // R + (i * 7 % 5 if N > 8 * R and 0 < i < R else 0) for i in range(R)} | {N})
    counts = [b - a for a, b in zip(cuts[:-1], cuts[1:])]
    return counts, [-1 if case["bare"] and i % 9 == 4 else (i * 5 + i // E) % E for i in range(len(counts))]


def _heavy(shape, gen, dtype=torch.float32):
    """Normal entries in rows whose size varies by a factor of a few, as hidden rows, keys and values do."""
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)
    x *= torch.exp(0.7 * torch.randn(shape[:-1] + (1,), generator=gen, device=DEV))
    return x.to(dtype)


def _pow2(e):
    """2^e in 32 bits for whole numbers within the normal range."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x):
    """(codes, scale bytes) of rows x [..., d]: the smallest power of two that brings them within 448."""
    amax = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(-60, 60)
    e = torch.where(amax == 0, torch.full_like(e, -60), e)
    return (x * _pow2(-e)).to(torch.float8_e4m3fn), (e + 127).squeeze(-1).to(torch.uint8)


def _int(a):
    return torch.tensor(a, dtype=torch.int32, device=DEV)


def _tables(lengths, page, order):
    """A block table that takes every request's pages from `order`, and the rest of `order`; -1 behind a request's last page."""
    per = [-(-t // page) for t in lengths]
    table = torch.full((len(per), max(per)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, p in enumerate(per):
        table[i, :p] = order[at:at + p]
        at += p
    return table, order[at:]


def _cache(case, pages, gen, dtype):
    """A filled pool of pages, and its scales in 8 bits."""
    Hkv, d, page = case["kv_heads"], case["dim"], case["page"]
    pool = torch.empty((pages, 2, Hkv, page, d), dtype=dtype, device=DEV)
    scales = torch.empty((pages, 2, Hkv, page), dtype=torch.uint8, device=DEV) if dtype == torch.float8_e4m3fn else None
    for p0 in range(0, pages, 1024):  # in parts: a user would not hold the 32-bit rows of a whole cache either
        x = _heavy((min(1024, pages - p0), 2, Hkv, page, d), gen)
        if scales is not None:
            pool[p0:p0 + 1024], scales[p0:p0 + 1024] = _quantise(x)
        else:
            pool[p0:p0 + 1024] = x.to(dtype)
    return pool, scales


def _received(shape, gen):
    """Sums of weights as steps leave them: a few keys hold most, many hold next to nothing, some nothing at all; every other head's
    are coarse, so that keys tie."""
    x = torch.exp(1.5 * torch.randn(shape, generator=gen, device=DEV) - 5)
    x[torch.rand(shape, generator=gen, device=DEV) < 0.05] = 0.0
    x[:, ::2] = x[:, ::2].to(torch.bfloat16).float()
    return x


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    st = {"case": case, "status": torch.zeros(1, dtype=torch.int32, device=DEV)}
    return {"weights": _prepare_weights, "choose": _prepare_choose, "compact": _prepare_compact, "adapt": _prepare_adapt}[case["kind"]](case, seed, gen, st)


def _prepare_weights(case, seed, gen, st):
    n, held = _lengths(case)
    R, N, Hq, Hkv, d = len(n), sum(n), case["heads"], case["kv_heads"], case["dim"]
    total = [a + b for a, b in zip(n, held)]
    firsts = [sum(n[:i]) for i in range(R + 1)]
    pages = sum(-(-t // case["page"]) for t in total)
    st["table"], _ = _tables(total, case["page"], torch.randperm(pages, generator=gen, device=DEV).to(torch.int32))
    st["req"] = torch.repeat_interleave(torch.arange(R, device=DEV), torch.tensor(n, device=DEV))
    st["within"] = torch.arange(N, device=DEV) - torch.tensor(firsts[:-1], device=DEV)[st["req"]]
    st["positions"] = (st["within"] + torch.tensor(held, device=DEV)[st["req"]]).to(torch.int32)
    st["cu_q"], st["longest"], st["max_kv"] = _int(firsts), max(n), max(total)
    st["pages"], st["scales"] = _cache(case, pages, gen, torch.bfloat16 if case["cache"] == "bfloat16" else torch.float8_e4m3fn)
    st["q"] = (1.5 * torch.randn((N, Hq, d), generator=gen, device=DEV)).to(torch.bfloat16)
    st["scale"] = d ** -0.5
    st["sink"] = torch.randn(Hq, generator=gen, device=DEV) if case["sink"] else None
    st["slopes"] = 2.0 ** (-8.0 * torch.arange(1, Hq + 1, device=DEV, dtype=torch.float32) / Hq) if case["slopes"] else None
    # what the steps before have left
    st["sums"] = _received((R, Hkv, max(total)), gen)
    return st


def _prepare_choose(case, seed, gen, st):
    lengths = _shares(case, 1)
    st["lengths"], st["keep"] = _int(lengths), _int([case["keep"]] * len(lengths))
    st["sums"] = _received((len(lengths), case["kv_heads"], max(lengths)), gen)
    st["width"] = min(case["keep"], max(lengths))
    return st


def _prepare_compact(case, seed, gen, st):
    lengths, Hkv, page = _shares(case, 1), case["kv_heads"], case["page"]
    R, kept = len(lengths), [min(case["keep"], t) for t in lengths]
    pages = sum(-(-t // page) for t in lengths) + sum(-(-t // page) for t in kept)
    st["table"], rest = _tables(lengths, page, torch.randperm(pages, generator=gen, device=DEV).to(torch.int32))
    st["into"], _ = _tables(kept, page, rest)
    st["pages"], st["scales"] = _cache(case, pages, gen, {"bfloat16": torch.bfloat16, "float8": torch.float8_e4m3fn, "float32": torch.float32}[case["cache"]])
    st["sums"] = _received((R, Hkv, max(lengths)), gen)
    st["sums_out"] = torch.zeros((R, Hkv, max(lengths)), device=DEV)
    # every head of every request keeps places of its own, in order
    places = torch.full((R, Hkv, max(kept)), -1, dtype=torch.int32, device=DEV)
    for r, (t, m) in enumerate(zip(lengths, kept)):
        places[r, :, :m] = torch.rand((Hkv, t), generator=gen, device=DEV).topk(m, -1).indices.sort(-1).values.to(torch.int32)
    st["places"], st["counts"] = places, _int(kept)
    return st


def _prepare_adapt(case, seed, gen, st):
    counts, adapters = _row_counts(case)
    N, E, r, K, No = case["rows"], case["adapters"], case["rank"], case["k"], case["n"]
    dtype, out_dtype = getattr(torch, case["dtype"]), getattr(torch, case["out_dtype"])
    st["of_row"] = [e for c, e in zip(counts, adapters) for _ in range(c)]
    st["e"] = torch.tensor(st["of_row"], device=DEV)
    st["x"] = _heavy((N, K), gen, dtype)
    st["a"] = (torch.randn((E, r, K), generator=gen, device=DEV) * K ** -0.5).to(dtype)
    st["b"] = (torch.randn((E, No, r), generator=gen, device=DEV) * r ** -0.5).to(dtype)
    st["y"] = _heavy((N, No), gen, out_dtype)
    st["scale"] = 0.5 + torch.rand(E, generator=gen, device=DEV)
    st["ranks"] = None
    if case["mixed_ranks"]:  # adapters of smaller rank lie padded with zeros
        ranks = [max(1, r >> (e % 3)) for e in range(E)]
        st["ranks"] = _int(ranks)
        behind = torch.arange(r, device=DEV)[None] >= st["ranks"][:, None]
        st["a"].masked_fill_(behind[:, :, None], 0)
        st["b"].masked_fill_(behind[:, None], 0)
    # the step's plan: made once, used by every layer's projections
    st["plan"] = _k().adapter_plan(st["of_row"], E) if own else None
    return st


# -------------------------------------------------------------------------------------------------- one pass of each
def run(st):
    kind = st["case"]["kind"]
    if own:
        return {"weights": _own_weights, "choose": _own_choose, "compact": _own_compact, "adapt": _own_adapt}[kind](st)
    return {"weights": _plain_weights, "choose": _plain_choose, "compact": _plain_compact, "adapt": _plain_adapt}[kind](st)


def _own_weights(st):
    case = st["case"]
    out = torch.empty_like(st["sums"])
    _k().attention_weights(st["q"], st["pages"], st["table"], st["cu_q"], st["positions"], out, st["scale"], case["chunk"], case["window"], case["temper"],
                           FLOOR, st["status"], st["max_kv"], st["longest"], scales=st["scales"], sink=st["sink"], slopes=st["slopes"], softcap=case["cap"],
                           add=st["sums"])
    return out


def _own_choose(st):
    case = st["case"]
    R, Hkv, _ = st["sums"].shape
    places = torch.empty((R, Hkv, st["width"]), dtype=torch.int32, device=st["sums"].device)
    counts = torch.empty(R, dtype=torch.int32, device=st["sums"].device)
    _k().kv_choose(st["sums"], st["lengths"], st["keep"], places, counts, st["status"], first=case["first"], recent=case["recent"])
    return {"places": places, "counts": counts}


def _moved(st):
    """The pool that holds the rows moved: codes of 8 bits as the whole numbers that they are, since rows move bit for bit."""
    if st["scales"] is None:
        return {"pages": st["pages"], "sums": st["sums_out"]}
    return {"pages": st["pages"].view(torch.uint8), "scales": st["scales"], "sums": st["sums_out"]}


def _own_compact(st):
    _k().kv_compact(st["pages"], st["table"], st["places"], st["counts"], st["status"], into=st["into"], scales=st["scales"], sums=st["sums"],
                    sums_out=st["sums_out"])
    return _moved(st)


def _own_adapt(st):
    out = torch.empty_like(st["y"])
    _k().adapter_add(st["x"], st["a"], st["b"], st["plan"], st["y"], out, scale=st["scale"], ranks=st["ranks"])
    return out


def _plain_weights(st):
    case = st["case"]
    R, L, T = st["table"].shape[0], st["max_kv"], st["longest"]
    Hq, Hkv, d = case["heads"], case["kv_heads"], case["dim"]
    G, req, within = Hq // Hkv, st["req"], st["within"]
    # every request's keys side by side, as the block table has them: [R, Hkv, L, d]
    table = st["table"].clamp(min=0).long()
    if st["scales"] is None:
        k = st["pages"][:, 0][table].float()
    else:
        k = st["pages"].view(torch.uint8)[:, 0][table].view(torch.float8_e4m3fn).float() * _pow2(st["scales"][:, 0][table].int().unsqueeze(-1) - 127)
    k = k.transpose(1, 2).flatten(2, 3)[:, :, :L]
    q = torch.zeros((R, T, Hq, d), device=k.device)
    q[req, within] = st["q"].float()
    pos = torch.full((R, T), -1, device=k.device)
    pos[req, within] = st["positions"].long()
    s = torch.einsum("rthgd,rhld->rhgtl", q.view(R, T, Hkv, G, d), k) * st["scale"]
    if case["temper"]:
        s = s * (1 + case["temper"] * torch.log1p(torch.floor((pos.float() + 1) / FLOOR)))[:, None, None, :, None]
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    place = torch.arange(L, device=k.device)
    lo = torch.zeros_like(pos)
    if case["chunk"]:
        lo = pos - pos % case["chunk"]
    if case["window"]:
        lo = torch.maximum(lo, pos - case["window"] + 1)
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, Hkv, G, 1, 1) * (pos[..., None] - place)[:, None, None]
    seen = (place <= pos[..., None]) & (place >= lo[..., None]) & (pos >= 0)[..., None]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    if st["sink"] is not None:
        m = torch.maximum(m, st["sink"].view(1, Hkv, G, 1, 1))
    m = m.clamp(min=-1e30)  # rows that see nothing
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    if st["sink"] is not None:
        total = total + torch.exp(st["sink"].view(1, Hkv, G, 1, 1) - m)
    return st["sums"] + (e / total.clamp(min=1e-38)).sum((2, 3))


def _plain_choose(st):
    case = st["case"]
    W = st["sums"].shape[2]
    place = torch.arange(W, device=st["sums"].device)
    length = st["lengths"].long()[:, None, None]
    n = torch.minimum(st["keep"].long()[:, None, None], length)
    recent = n.clamp(max=case["recent"])
    first = (n - recent).clamp(max=case["first"])
    # two stable sorts: by the sum, then by whether a place is kept whatever its sum, or does not exist
    rank = torch.where(place >= length, 2, torch.where((place < first) | (place >= length - recent), 0, 1)).expand(st["sums"].shape)
    order = st["sums"].sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, rank.gather(-1, order).sort(dim=-1, stable=True).indices)[..., :st["width"]]
    at = torch.arange(st["width"], device=place.device)
    kept = torch.where(at < n, order, W).sort(-1).values
    return {"places": torch.where(at < n, kept, -1).to(torch.int32), "counts": n[:, 0, 0].to(torch.int32)}


def _plain_compact(st):
    Hkv, page = st["case"]["kv_heads"], st["case"]["page"]
    r, h, i = (st["places"] >= 0).nonzero(as_tuple=True)
    j = st["places"][r, h, i].long()
    src, dst = st["table"][r, j // page].long(), st["into"][r, i // page].long()
    bits = st["pages"].view(torch.uint8)
    bits[dst, :, h, i % page] = bits[src, :, h, j % page]
    if st["scales"] is not None:
        st["scales"][dst, :, h, i % page] = st["scales"][src, :, h, j % page]
    st["sums_out"].zero_()
    st["sums_out"][r, h, i] = st["sums"][r, h, j]
    return _moved(st)


def _plain_adapt(st):
    """Both products over all adapters side by side: a row's own part of the first one is kept, the others' are zeros in the second."""
    N, (E, r, K) = st["x"].shape[0], st["a"].shape
    low = (st["x"].float() @ st["a"].float().view(E * r, K).T).view(N, E, r)
    mine = (st["e"][:, None] == torch.arange(E, device=low.device)).float() * st["scale"]
    more = (low * mine[:, :, None]).view(N, E * r) @ st["b"].float().transpose(1, 2).reshape(E * r, -1)
    return (st["y"].float() + more).to(st["y"].dtype)


# ---------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    """Bytes: of the cache each visible key (kept row) of every request once, weights of the adapters in use once, rows in and out."""
    if case["kind"] == "adapt":
        counts, adapters = _row_counts(case)
        size, out = (4 if case["dtype"] == "float32" else 2), (4 if case["out_dtype"] == "float32" else 2)
        rank = lambda e: max(1, case["rank"] >> (e % 3)) if case["mixed_ranks"] else case["rank"]  # noqa: E731
        weights = sum(rank(e) for e in set(adapters) - {-1}) * (case["k"] + case["n"]) * size
        rows = sum(c for c, e in zip(counts, adapters) if e >= 0)
        flops = 2 * sum(c * rank(e) for c, e in zip(counts, adapters) if e >= 0) * (case["k"] + case["n"])
        return {"bytes": weights + rows * case["k"] * size + 2 * case["rows"] * case["n"] * out, "flops": flops}
    if case["kind"] == "choose":
        lengths = _shares(case, 1)
        return {"bytes": 4 * case["kv_heads"] * sum(t + min(t, case["keep"]) for t in lengths), "flops": case["kv_heads"] * sum(lengths)}
    Hkv, d = case["kv_heads"], case["dim"]
    if case["kind"] == "compact":
        lengths = _shares(case, 1)
        row = 2 * (d + 1 if case["cache"] == "float8" else 2 * d if case["cache"] == "bfloat16" else 4 * d)
        return {"bytes": Hkv * sum(min(t, case["keep"]) * (2 * row + 8) for t in lengths) + 4 * Hkv * len(lengths) * max(lengths), "flops": 0}
    n, held = _lengths(case)
    row = Hkv * (d + 1 if case["cache"] == "float8" else 2 * d)
    first = lambda p: max(p - p % case["chunk"] if case["chunk"] else 0, p - case["window"] + 1 if case["window"] else 0, 0)  # noqa: E731
    keys = sum(c + m - first(c) for m, c in zip(n, held))
    pairs = sum(sum(p + 1 - first(p) for p in range(c, c + m)) for m, c in zip(n, held))
    top = max(a + b for a, b in zip(n, held))
    return {"bytes": keys * row + 2 * sum(n) * case["heads"] * d + 8 * len(n) * Hkv * top, "flops": 2 * d * case["heads"] * pairs}


# --------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    if case["kind"] == "choose":
        return None  # places are whole numbers
    return {"weights": _exact_weights, "compact": _exact_compact, "adapt": _exact_adapt}[case["kind"]](prepare(case, seed))


def _two_to(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_weights(st):
    """Request by request, head group by head group."""
    case = st["case"]
    n, held = _lengths(case)
    G, page = case["heads"] // case["kv_heads"], case["page"]
    out = st["sums"].double()
    f = 0
    for r, (m, c) in enumerate(zip(n, held)):
        L = m + c
        key = torch.arange(L, device=out.device)
        where, at = st["table"][r].long()[key // page], key % page
        p = st["positions"][f:f + m].double()
        lo = torch.zeros(m, dtype=torch.float64, device=out.device)
        if case["chunk"]:
            lo = torch.floor(p / case["chunk"]) * case["chunk"]
        if case["window"]:
            lo = torch.maximum(lo, p - case["window"] + 1)
        hidden = (key[None] > p[:, None]) | (key[None] < lo[:, None])
        for h in range(case["kv_heads"]):
            if st["scales"] is None:
                k = st["pages"][where, 0, h, at].double()
            else:
                k = st["pages"].view(torch.uint8)[where, 0, h, at].view(torch.float8_e4m3fn).double() * _two_to(st["scales"][where, 0, h, at].long() - 127)[:, None]
            for g in range(h * G, h * G + G):
                s = torch.matmul(st["q"][f:f + m, g].double(), k.T) * st["scale"]
                if case["temper"]:
                    s = s * (1 + case["temper"] * torch.log1p(torch.floor((p + 1) / FLOOR)))[:, None]
                if case["cap"]:
                    s = case["cap"] * torch.tanh(s / case["cap"])
                if st["slopes"] is not None:
                    s = s - st["slopes"][g].double() * (p[:, None] - key[None])
                s = torch.where(hidden, -math.inf, s)
                lse = torch.logsumexp(s, -1)
                if st["sink"] is not None:
                    lse = torch.logaddexp(lse, st["sink"][g].double())
                out[r, h, :L] += torch.exp(s - lse.clamp(min=-1e300)[:, None]).sum(0)
        f += m
    return out


def _exact_compact(st):
    moved = torch.zeros_like(st["sums_out"], dtype=torch.float64)
    for r, m in enumerate(st["counts"].tolist()):
        moved[r, :, :m] = torch.take_along_dim(st["sums"][r].double(), st["places"][r, :, :m].long(), -1)
    out = {"pages": None, "sums": moved}
    if st["scales"] is not None:
        out["scales"] = None
    return out


def _exact_adapt(st):
    """Adapter by adapter."""
    out = st["y"].double()
    e = st["e"]
    for i in range(st["a"].shape[0]):
        mine = e == i
        if bool(mine.any()):
            low = torch.einsum("nk,rk->nr", st["x"][mine].double(), st["a"][i].double())
            out[mine] += st["scale"][i].double() * torch.einsum("nr,mr->nm", low, st["b"][i].double())
    return out
