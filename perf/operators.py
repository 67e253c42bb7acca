"""What the 8-bit cache and the attention over it are measured by: the calls that a program around this engine makes.

Three operators over a paged cache (pages of keys and values, found through a block table):

* ``store``: a step's keys and values are written in 8 bits (e4m3 codes, one power of two per token, head and plane) and read
  back as the values they stand for.  ``form`` "rope": from projected rows, with the rotation and the q/k norm in the same
  pass; "rows": from encoded keys and values.
* ``attend``: causal grouped-query attention over such a cache, for a step's single tokens and its prompt portions.
* ``tree``: attention of a request's drafted tokens, each seeing the cached keys and its own ancestors, over a bfloat16 or an
  8-bit cache.

A stored row: amax = max |x|, e = the smallest whole number with amax <= 448 * 2^e, at least -60; codes = x * 2^-e rounded to
e4m3 (ties to even), scale byte = e + 127.  Plain forms are torch in 32 bits; ``exact`` restates them in 64."""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
FLOOR = 8192.0  # positions between two steps of the attention temperature
EPS = 1e-5
CUT = 128  # tokens of a prompt portion that a work item holds
NO_POSITION = -1


def _k():
    from jax_llm_examples_b200.kernels import api

    return api


# ------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a decode step of a serving batch: split-K partials of the projection in, one row a request
        {"name": "store_decode_64", "kind": "store", "form": "rope", "tokens": 64, "requests": 64, "heads": 40, "kv_heads": 8, "dim": 128,
         "page": 64, "start": 8000, "splits": 4, "dtype": "float32", "norm": True},
        # a long prompt portion's projected rows
        {"name": "store_prompt_4096", "kind": "store", "form": "rope", "tokens": 4096, "requests": 1, "heads": 40, "kv_heads": 8, "dim": 128,
         "page": 64, "start": 0, "splits": 1, "dtype": "bfloat16", "norm": True},
        # rows that another encoding made, in 32 bits, small heads, small pages, ragged
        {"name": "store_rows_1777", "kind": "store", "form": "rows", "tokens": 1777, "requests": 5, "heads": 4, "kv_heads": 4, "dim": 64,
         "page": 16, "start": 300, "splits": 1, "dtype": "float32", "norm": False},
        # one chat session: the latency of a token
        {"name": "attend_one", "kind": "attend", "requests": 1, "tokens": 1, "portions": 0, "context": 700, "ragged": False, "heads": 40,
         "kv_heads": 8, "dim": 128, "page": 64, "chunk": 0, "window": 0, "temper": 0.0, "cap": 0.0, "sink": False, "slopes": False},
        # serving batches of ragged sessions: small and long, large
        {"name": "attend_8_long", "kind": "attend", "requests": 8, "tokens": 1, "portions": 0, "context": 30001, "ragged": True, "heads": 40,
         "kv_heads": 8, "dim": 128, "page": 64, "chunk": 0, "window": 0, "temper": 0.1, "cap": 0.0, "sink": False, "slopes": False},
        {"name": "attend_64", "kind": "attend", "requests": 64, "tokens": 1, "portions": 0, "context": 8192, "ragged": True, "heads": 40,
         "kv_heads": 8, "dim": 128, "page": 64, "chunk": 0, "window": 0, "temper": 0.0, "cap": 0.0, "sink": False, "slopes": False},
        # a prompt portion behind cached tokens, in the scheduler's default size
        {"name": "attend_portion_2048", "kind": "attend", "requests": 1, "tokens": 2048, "portions": 1, "context": 1500, "ragged": False,
         "heads": 40, "kv_heads": 8, "dim": 128, "page": 64, "chunk": 8192, "window": 0, "temper": 0.0, "cap": 0.0, "sink": False, "slopes": False},
        # short portions beside single tokens, small heads, a window, a sink and capped scores
        {"name": "attend_mixed_64", "kind": "attend", "requests": 9, "tokens": 333, "portions": 3, "context": 5000, "ragged": True,
         "heads": 16, "kv_heads": 4, "dim": 64, "page": 48, "chunk": 0, "window": 1024, "temper": 0.0, "cap": 30.0, "sink": True, "slopes": False},
        # a few drafted tokens of one session
        {"name": "tree_one_8", "kind": "tree", "cache": "bfloat16", "requests": 1, "tokens": 8, "context": 900, "ragged": False, "heads": 40,
         "kv_heads": 8, "dim": 128, "page": 64, "chunk": 0, "window": 0, "temper": 0.0, "cap": 0.0, "sink": False, "slopes": False},
        # a serving batch with a tree each, over either cache
        {"name": "tree_8_32", "kind": "tree", "cache": "bfloat16", "requests": 8, "tokens": 32, "context": 8192, "ragged": True, "heads": 40,
         "kv_heads": 8, "dim": 128, "page": 64, "chunk": 0, "window": 0, "temper": 0.0, "cap": 0.0, "sink": False, "slopes": False},
        {"name": "tree_16_64_8bit", "kind": "tree", "cache": "float8", "requests": 16, "tokens": 64, "context": 12000, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "chunk": 0, "window": 0, "temper": 0.0, "cap": 0.0, "sink": True, "slopes": False},
        # small heads without groups, a distance bias behind a window
        {"name": "tree_4_13_64", "kind": "tree", "cache": "float8", "requests": 4, "tokens": 13, "context": 2500, "ragged": True, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16, "chunk": 0, "window": 2000, "temper": 0.0, "cap": 0.0, "sink": False, "slopes": True},
    ]


def _log(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# query heads, key/value heads, head size: this package's presets and their neighbours, groups of 1 to 16
HEADS = [(40, 8, 128), (32, 8, 128), (16, 4, 128), (16, 4, 64), (12, 12, 64), (16, 2, 128), (32, 2, 128), (6, 3, 64), (24, 8, 128), (8, 8, 128)]


def draw(rng):
    """Steps of serving batches: rows to store, single tokens and portions, drafted trees, of every size up to the listed ones."""
    kind = rng.choice(["store", "attend", "attend", "tree", "tree"])
    heads, kv_heads, dim = rng.choice(HEADS)
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 48, 64, 64, 64, 128])}
    if kind == "store":
        tokens = _log(rng, 1, 4096)
        form = rng.choice(["rope", "rope", "rows"])
        splits = rng.choice([1, 2, 5]) if form == "rope" and tokens <= 256 else 1
        case |= {"form": form, "tokens": tokens, "requests": min(tokens, _log(rng, 1, 64)), "start": _log(rng, 1, 100000), "splits": splits,
                 "dtype": "float32" if splits > 1 else rng.choice(["float32", "bfloat16"]), "norm": form == "rope" and rng.random() < 0.5}
        return case
    context = _log(rng, 1, 32768)
    mask = rng.choice(["all", "all", "all", "chunk", "window"])
    case |= {"ragged": rng.random() < 0.7, "chunk": _log(rng, 64, 8192) if mask == "chunk" else 0, "window": _log(rng, 16, 4096) if mask == "window" else 0,
             "temper": rng.choice([0.0, 0.0, 0.1]), "cap": rng.choice([0.0, 0.0, 0.0, 30.0]), "sink": rng.random() < 0.3, "slopes": rng.random() < 0.2}
    if kind == "tree":
        tokens = _log(rng, 1, 96)
        most = max(1, min(32, int(1.2e7 // (tokens * max(context, 256) * heads // 40 + 1))))
        case |= {"cache": rng.choice(["bfloat16", "float8"]), "tokens": tokens, "requests": _log(rng, 1, most), "context": context}
        return case
    if rng.random() < 0.5:
        most = max(1, min(128, 500000 // context))
        case |= {"tokens": 1, "portions": 0, "requests": _log(rng, 1, most), "context": context}
        return case
    tokens = _log(rng, 2, 2048)
    context = min(context, 4000)
    portions = rng.randint(1, max(1, min(4, 2048 // tokens)))
    case |= {"tokens": tokens, "portions": portions, "requests": portions + rng.choice([0, 0, 1, 7 if tokens <= 256 else 2]), "context": context}
    return case


# ----------------------------------------------------------------------------------------------------- the inputs
def _lengths(case):
    """(tokens each request brings, tokens it held before): host lists."""
    R, T = case["requests"], case["tokens"]
    if case["kind"] == "store":
        n = [T // R + (i < T % R) for i in range(R)]
        return n, [case["start"] + 37 * i for i in range(R)]
    held = [max(0, case["context"] - (i * 2654435761 % 1000 * case["context"] // 2000 if case["ragged"] and i else 0)) for i in range(R)]
    if case["kind"] == "tree":
        n = [max(1, T - (i % 4 if case["ragged"] else 0)) for i in range(R)]
    else:
        n = [max(1, T - (i * 5 if case["ragged"] else 0)) if i < case["portions"] else 1 for i in range(R)]
        held = [c - 1 if m == 1 and c > 0 else c for c, m in zip(held, n)]
    return n, held


def _heavy(shape, gen, dtype=torch.float32):
    """Normal entries in rows whose size varies by a factor of a few, as projected keys and values do."""
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)
    x *= torch.exp(0.7 * torch.randn(shape[:-1] + (1,), generator=gen, device=DEV))
    return x.to(dtype)


def _pow2(e):
    """2^e in 32 bits for whole numbers within the normal range: a power function may be a unit off, and would break ties."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x):
    """(codes, scale bytes) of rows x [..., d]: see the module's text."""
    amax = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(-60, 60)
    e = torch.where(amax == 0, torch.full_like(e, -60), e)
    codes = (x * _pow2(-e)).to(torch.float8_e4m3fn)
    return codes, (e + 127).squeeze(-1).to(torch.uint8)


def _int(a):
    return torch.tensor(a, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    n, held = _lengths(case)
    R, N, page = len(n), sum(n), case["page"]
    Hq, Hkv, d = case["heads"], case["kv_heads"], case["dim"]
    total = [a + b for a, b in zip(n, held)]
    per = [-(-t // page) for t in total]
    width = max(per)
    firsts = [sum(n[:i]) for i in range(R + 1)]
    st = {"case": case, "page": page}
    # every request's pages, scattered over the pool; entries behind a request's last page name none
    order = torch.randperm(sum(per), generator=gen, device=DEV).to(torch.int32)
    table = torch.full((R, width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, p in enumerate(per):
        table[i, :p] = order[at:at + p]
        at += p
    P = sum(per)
    st["table"] = table
    st["req"] = torch.repeat_interleave(torch.arange(R, device=DEV), torch.tensor(n, device=DEV)).to(torch.int32)
    within = torch.arange(N, device=DEV) - torch.tensor(firsts[:-1], device=DEV)[st["req"].long()]
    st["within"] = within
    st["places"] = (within + torch.tensor(held, device=DEV)[st["req"].long()]).to(torch.int32)
    st["status"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    st["n"], st["longest"], st["max_kv"] = N, max(n), max(total)
    if case["kind"] == "store":
        dtype = getattr(torch, case["dtype"])
        st["pages"] = torch.zeros((P, 2, Hkv, page, d), dtype=torch.float8_e4m3fn, device=DEV)
        st["scales"] = torch.zeros((P, 2, Hkv, page), dtype=torch.uint8, device=DEV)
        if case["form"] == "rows":
            st["k"], st["v"] = _heavy((N, Hkv, d), gen, dtype), _heavy((N, Hkv, d), gen, dtype)
        else:
            s = case["splits"]
            rows = _heavy((s, N, Hq + 2 * Hkv, d) if s > 1 else (N, Hq + 2 * Hkv, d), gen) / math.sqrt(s)
            st["qkv"] = rows.flatten(-2).to(dtype).contiguous()
            st["inv_freq"] = 500000.0 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float32) / d)
        return st
    # a filled cache, and queries whose softmax is spread as a trained head's
    st["scale"] = d ** -0.5
    bits8 = case["kind"] == "attend" or case["cache"] == "float8"
    pages = torch.empty((P, 2, Hkv, page, d), dtype=torch.float8_e4m3fn if bits8 else torch.bfloat16, device=DEV)
    scales = torch.empty((P, 2, Hkv, page), dtype=torch.uint8, device=DEV) if bits8 else None
    for p0 in range(0, P, 1024):  # in parts: the 32-bit rows of a whole cache would not be held by a user either
        x = _heavy((min(1024, P - p0), 2, Hkv, page, d), gen)
        if bits8:
            pages[p0:p0 + 1024], scales[p0:p0 + 1024] = _quantise(x)
        else:
            pages[p0:p0 + 1024] = x.to(torch.bfloat16)
    st["pages"], st["scales"] = pages, scales
    st["q"] = (1.5 * torch.randn((N, Hq, d), generator=gen, device=DEV)).to(torch.bfloat16)
    st["sink"] = torch.randn(Hq, generator=gen, device=DEV) if case["sink"] else None
    st["slopes"] = 2.0 ** (-8.0 * torch.arange(1, Hq + 1, device=DEV, dtype=torch.float32) / Hq) if case["slopes"] else None
    st["cu_q"], st["q_start"] = _int(firsts), _int(held)
    if case["kind"] == "tree":
        # each drafted token's parent is an earlier one or the last cached token; a token sees its ancestors and itself
        words = -(-max(n) // 32)
        depth, bits = torch.zeros(N, dtype=torch.int32), torch.zeros((N, words), dtype=torch.int64)
        pick = torch.rand(N, generator=torch.Generator().manual_seed(int(seed) + 1))
        for i in range(R):
            for j in range(n[i]):
                row = firsts[i] + j
                parent = int(pick[row] * (j + 1)) - 1 if j else NO_POSITION
                if parent >= 0:
                    depth[row] = depth[firsts[i] + parent] + 1
                    bits[row] = bits[firsts[i] + parent]
                bits[row, j // 32] |= 1 << (j % 32)
        st["masks"] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32).to(DEV)
        st["positions"] = (torch.tensor(held)[st["req"].cpu().long()] + depth).to(torch.int32).to(DEV)
        st["items"], st["n_items"], st["max_count"] = _int([[f, m] for f, m in zip(firsts, n)]), R, max(n)
        return st
    st["positions"] = st["places"]
    # the step's plan: portions cut into work items, and the rows of the requests that bring one token
    items = [[f + o, min(CUT, m - o)] for f, m in zip(firsts, n) if m > 1 for o in range(0, m, CUT)][::-1]
    rows = [f for f, m in zip(firsts, n) if m == 1]
    st["items"], st["n_items"], st["max_count"] = (_int(items) if items else None), len(items), max([c for _, c in items], default=1)
    st["rows"], st["n_rows"] = (_int(rows) if rows and items else None), len(rows)
    return st


# -------------------------------------------------------------------------------------------------- one pass of each
def run(st):
    case = st["case"]
    if own:
        return {"store": _own_store, "attend": _own_attend, "tree": _own_tree}[case["kind"]](st)
    return _plain_store(st) if case["kind"] == "store" else _plain_attention(st)


def _own_store(st):
    K, case = _k(), st["case"]
    d, Hq, Hkv, N = case["dim"], case["heads"], case["kv_heads"], st["n"]
    out = {}
    if case["form"] == "rows":
        dtype = st["k"].dtype
        K.kv_store_fp8(st["k"], st["v"], st["pages"], st["scales"], st["table"], st["req"], st["places"], st["status"])
    else:
        dtype = torch.bfloat16
        out["q"] = torch.empty((N, Hq, d), dtype=dtype, device=st["qkv"].device)
        K.rope_kv_store_fp8(st["qkv"], out["q"], st["pages"], st["scales"], st["table"], st["req"], st["places"], st["inv_freq"], case["norm"], EPS,
                            Hq, Hkv, d, st["status"], case["splits"])
    out["k"], out["v"] = (torch.empty((N, Hkv, d), dtype=dtype, device=st["pages"].device) for _ in range(2))
    K.kv_load_fp8(st["pages"], st["scales"], st["table"], st["req"], st["places"], out["k"], out["v"], st["status"])
    return out


def _own_attend(st):
    K, case = _k(), st["case"]
    out = torch.empty_like(st["q"])
    head = (st["q"], st["pages"], st["scales"], st["table"], st["req"], st["positions"], out, st["scale"], case["chunk"], case["window"],
            case["temper"], FLOOR, st["status"], st["max_kv"])
    tail = {"sink": st["sink"], "slopes": st["slopes"], "softcap": case["cap"]}
    if st["n_items"]:
        K.attention_fp8(*head, items=st["items"], n_items=st["n_items"], max_count=st["max_count"], **tail)
    if st["n_rows"]:
        K.attention_fp8(*head, rows=st["rows"], n_rows=st["n_rows"], **tail)
    return out


def _own_tree(st):
    K, case = _k(), st["case"]
    out = torch.empty_like(st["q"])
    K.attention_tree(st["q"], st["pages"], st["table"], st["req"], st["positions"], st["cu_q"], st["q_start"], st["masks"], out, st["scale"],
                     case["chunk"], case["window"], case["temper"], FLOOR, st["status"], st["max_kv"], st["items"], st["n_items"], st["max_count"],
                     scales=st["scales"], sink=st["sink"], slopes=st["slopes"], softcap=case["cap"])
    return out


def _plain_store(st):
    case = st["case"]
    d, Hq, Hkv, N = case["dim"], case["heads"], case["kv_heads"], st["n"]
    out = {}
    if case["form"] == "rows":
        k, v = st["k"].float(), st["v"].float()
        dtype = st["k"].dtype
    else:
        x = st["qkv"].float()
        x = (x.sum(0) if case["splits"] > 1 else x).view(N, Hq + 2 * Hkv, d)
        qk, v = x[:, :Hq + Hkv], x[:, Hq + Hkv:]
        angle = st["places"].double()[:, None] * st["inv_freq"].double()  # far positions: 32 bits would lose the turn's fraction
        c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
        a, b = qk[..., 0::2], qk[..., 1::2]
        qk = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
        if case["norm"]:
            qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS)
        dtype = torch.bfloat16
        out["q"], k = qk[:, :Hq].to(dtype).contiguous(), qk[:, Hq:]
    page, at = st["table"][st["req"].long(), (st["places"] // st["page"]).long()].long(), (st["places"] % st["page"]).long()
    codes, scales = _quantise(torch.stack([k, v], 1))
    st["pages"].view(torch.uint8)[page, :, :, at] = codes.view(torch.uint8)
    st["scales"][page, :, :, at] = scales
    codes, scales = st["pages"].view(torch.uint8)[page, :, :, at].view(torch.float8_e4m3fn), st["scales"][page, :, :, at]
    back = (codes.float() * _pow2(scales.int().unsqueeze(-1) - 127)).to(dtype)
    out["k"], out["v"] = back[:, 0].contiguous(), back[:, 1].contiguous()
    return out


def _plain_attention(st):
    case = st["case"]
    R, L, T, tree = st["table"].shape[0], st["max_kv"], st["longest"], case["kind"] == "tree"
    Hq, Hkv, d = case["heads"], case["kv_heads"], case["dim"]
    G, req, within = Hq // Hkv, st["req"].long(), st["within"]
    # every request's rows side by side, as the block table has them: [R, 2, Hkv, L, d]
    table = st["table"].clamp(min=0).long()
    kv = st["pages"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() if st["scales"] is not None else st["pages"][table].float()
    if st["scales"] is not None:
        kv = kv * _pow2(st["scales"][table].int().unsqueeze(-1) - 127)
    kv = kv.permute(0, 2, 3, 1, 4, 5).flatten(3, 4)
    q = torch.zeros((R, T, Hq, d), device=kv.device)
    q[req, within] = st["q"].float()
    pos = torch.full((R, T), NO_POSITION, device=kv.device)
    pos[req, within] = st["positions"].long()
    s = torch.einsum("rthgd,rhld->rhgtl", q.view(R, T, Hkv, G, d), kv[:, 0])[..., :L] * st["scale"]
    if case["temper"]:
        s = s * (1 + case["temper"] * torch.log1p(torch.floor((pos.float() + 1) / FLOOR)))[:, None, None, :, None]
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    place = torch.arange(L, device=kv.device).expand(R, L)
    lo = torch.zeros_like(pos)
    if case["chunk"]:
        lo = pos - pos % case["chunk"]
    if case["window"]:
        lo = torch.maximum(lo, pos - case["window"] + 1)
    if tree:
        base = st["q_start"].long()[:, None]
        j = (place - base).clamp(0, T - 1)  # which drafted token lies at the place
        key_pos = torch.where(place < base, place, pos.gather(1, j))
        words = torch.zeros((R, T, st["masks"].shape[1]), dtype=torch.int32, device=kv.device)
        words[req, within] = st["masks"]
        bit = (words.gather(2, (j // 32)[:, None].expand(R, T, L)) >> (j % 32)[:, None].int()) & 1
        drafted = (place >= base) & (place < base + (st["cu_q"][1:] - st["cu_q"][:-1]).long()[:, None])
        seen = (place < base)[:, None] | (drafted[:, None] & (bit == 1))
    else:
        key_pos = place
        seen = place[:, None] <= pos[..., None]
    seen = seen & (key_pos[:, None] >= lo[..., None]) & (pos >= 0)[..., None]
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, Hkv, G, 1, 1) * (pos[..., None] - key_pos[:, None])[:, None, None]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    if st["sink"] is not None:
        m = torch.maximum(m, st["sink"].view(1, Hkv, G, 1, 1))
    m = m.clamp(min=-1e30)  # rows that see nothing
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    if st["sink"] is not None:
        total = total + torch.exp(st["sink"].view(1, Hkv, G, 1, 1) - m)
    o = torch.einsum("rhgtl,rhld->rthgd", e, kv[:, 1, :, :L]) / total.clamp(min=1e-38).permute(0, 3, 1, 2, 4)
    return o.reshape(R, T, Hq, d)[req, within].to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    """Bytes: projected rows, queries and outputs once, and of the cache each visible row (and its scale) of every request once."""
    n, held = _lengths(case)
    Hq, Hkv, d = case["heads"], case["kv_heads"], case["dim"]
    N = sum(n)
    if case["kind"] == "store":
        size = 4 if case["dtype"] == "float32" else 2
        back = 2 * N * Hkv * d * (2 if case["form"] == "rope" else size)
        rows = case["splits"] * N * (Hq + 2 * Hkv) * d * size + N * Hq * d * 2 if case["form"] == "rope" else 2 * N * Hkv * d * size
        return {"bytes": rows + back + 2 * N * Hkv * (d + 1), "flops": 8 * N * (Hq + 2 * Hkv) * d}
    row = 2 * Hkv * (d + 1) if case["kind"] == "attend" or case["cache"] == "float8" else 2 * Hkv * d * 2
    keys = pairs = 0
    for m, c in zip(n, held):
        first = lambda p: max(p - p % case["chunk"] if case["chunk"] else 0, p - case["window"] + 1 if case["window"] else 0, 0)  # noqa: E731
        if case["kind"] == "tree":
            seen = c - min(first(c), c)
            keys += seen + m
            pairs += m * (seen + min(m, 6))
        else:
            keys += c + m - first(c)
            pairs += sum(p + 1 - first(p) for p in range(c, c + m))
    return {"bytes": keys * row + 4 * N * Hq * d, "flops": 4 * d * Hq * pairs}


# --------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return _exact_store(st) if case["kind"] == "store" else _exact_attention(st)


def _two_to(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _held_in_8(x):
    """What a row of 64-bit numbers is held as: the grid of e4m3 has 2^-9 below 2^-6, and eight steps in every octave above."""
    top = x.abs().max(-1, keepdim=True).values
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448)).clamp(-60, 60)
    e = torch.where(top > 448 * _two_to(e), e + 1, e)
    y = x / _two_to(e)
    octave = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    octave = torch.where(_two_to(octave + 1) <= y.abs(), octave + 1, octave)
    step = _two_to(octave - 3)
    return torch.round(y / step) * step * _two_to(e)


def _exact_store(st):
    case = st["case"]
    Hq, Hkv = case["heads"], case["kv_heads"]
    if case["form"] == "rows":
        return {"k": _held_in_8(st["k"].double()), "v": _held_in_8(st["v"].double())}
    x = st["qkv"].double()
    if case["splits"] > 1:
        x = x.sum(0)
    z = torch.view_as_complex(x.view(st["n"], Hq + 2 * Hkv, case["dim"] // 2, 2))
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=z.device), st["places"].double()[:, None] * st["inv_freq"].double())
    turned = torch.view_as_real(z[:, :Hq + Hkv] * turn[:, None]).flatten(-2)
    if case["norm"]:
        turned = turned * (turned.square().mean(-1, keepdim=True) + EPS).rsqrt()
    v = torch.view_as_real(z[:, Hq + Hkv:]).flatten(-2)
    return {"q": turned[:, :Hq], "k": _held_in_8(turned[:, Hq:]), "v": _held_in_8(v)}


def _exact_attention(st):
    """Request by request, head group by head group."""
    case = st["case"]
    n, held = _lengths(case)
    Hq, Hkv, d, page = case["heads"], case["kv_heads"], case["dim"], st["page"]
    G = Hq // Hkv
    out = torch.zeros((st["n"], Hq, d), dtype=torch.float64, device=st["q"].device)
    f = 0
    for r, (m, c) in enumerate(zip(n, held)):
        L = m + c
        rows = torch.arange(L, device=out.device)
        where, at = st["table"][r].long()[rows // page], rows % page
        p = st["positions"][f:f + m].double()
        lo = torch.zeros(m, dtype=torch.float64, device=out.device)
        if case["chunk"]:
            lo = torch.floor(p / case["chunk"]) * case["chunk"]
        if case["window"]:
            lo = torch.maximum(lo, p - case["window"] + 1)
        key = rows.double()
        if case["kind"] == "tree":
            key = torch.cat([key[:c], p])
            bits = torch.stack([(st["masks"][f:f + m, j // 32] >> (j % 32)) & 1 for j in range(m)], 1) == 1
            seen = torch.cat([torch.ones((m, c), dtype=torch.bool, device=out.device), bits], 1)
        else:
            seen = key[None] <= p[:, None]
        seen &= key[None] >= lo[:, None]
        for h in range(Hkv):
            if st["scales"] is None:
                k, v = st["pages"][where, 0, h, at].double(), st["pages"][where, 1, h, at].double()
            else:
                raw = st["pages"].view(torch.uint8)
                k, v = (raw[where, w, h, at].view(torch.float8_e4m3fn).double() * _two_to(st["scales"][where, w, h, at].long() - 127)[:, None] for w in (0, 1))
            q = st["q"][f:f + m, h * G:(h + 1) * G].double()
            s = torch.matmul(q.transpose(0, 1), k.T) * st["scale"]
            if case["temper"]:
                s = s * (1 + case["temper"] * torch.log1p(torch.floor((p + 1) / FLOOR)))[:, None]
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            if st["slopes"] is not None:
                s = s - st["slopes"][h * G:(h + 1) * G].double()[:, None, None] * (p[:, None] - key[None])
            s = torch.where(seen, s, -math.inf)
            if st["sink"] is not None:
                s = torch.cat([s, st["sink"][h * G:(h + 1) * G].double()[:, None, None].expand(G, m, 1)], -1)
            w = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)[..., :L]
            out[f:f + m, h * G:(h + 1) * G] = torch.matmul(w, v).transpose(0, 1)
        f += m
    return out
