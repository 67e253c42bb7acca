"""The 8-bit cache and the attention over rows at the ends of their format and their calls, against 64 bits (fp8_helpers.py)."""

import math

import pytest
import torch

from .fp8_helpers import Case, assert_close, hold

pytestmark = pytest.mark.gpu


def K():
    from jax_llm_examples_b200.kernels import api

    return api


FORMS = ["rule", "attention_rows", "attention_rows_tc", "attention_few"]  # the kernel by the sizes, or the one named


@pytest.fixture
def form(request, monkeypatch):
    rule = K().attention_rows_form
    if request.param != "rule":  # (the tcgen05 kernel where it can)
        monkeypatch.setattr(K(), "attention_rows_form",
                            lambda rows, page, aligned, *a: rule(rows, page, aligned, *a) if request.param == "attention_rows_tc" and (page % 16 or not aligned)
                            else request.param)
    return request.param


def _serve(c, mask=None, items=None, rows=None):
    """Holds the case to the bound of the kernel that serves these items (to be called before the case is asked for it)."""
    mask = mask or {}
    if c.masks is not None:
        items = items or c.items(max(c.n))
    most = items[2] if items is not None else 1
    n_items = items[1] if items is not None else (rows.numel() if rows is not None else c.N)
    seen = K()._keys_seen(max(a + b for a, b in zip(c.n, c.held)), mask.get("chunk", 0), mask.get("window", 0), most)
    aligned = c.scales is None or c.scales.data_ptr() % 16 == 0
    kernel = K().attention_rows_form(most * (c.Hq // c.Hkv), c.page, aligned, seen, n_items * c.Hkv, c.bits8)
    c.weights = 2.0 ** -11 if c.bits8 and kernel != "attention_rows_tc" else 2.0 ** -8
    return items


def _call(c, mask=None, items=None, out=None, rows=None, **kw):
    """The causal call over 8 bits or, where the case is a tree, the tree's."""
    mask, out = mask or {}, torch.full_like(c.q, 7.0) if out is None else out
    items = _serve(c, mask, items, rows)
    how = (c.scale, mask.get("chunk", 0), mask.get("window", 0), mask.get("temper", 0.0), mask.get("floor", 1.0), c.status,
           max(a + b for a, b in zip(c.n, c.held)))
    if c.masks is not None:
        K().attention_tree(c.q, c.pages, c.table, c.req, c.positions, c.cu_q, c.q_start, c.masks, out, *how, *items, scales=c.scales, **kw)
    else:
        if items is not None:
            kw |= dict(items=items[0], n_items=items[1], max_count=items[2])
        if rows is not None:
            kw |= dict(rows=rows, n_rows=rows.numel())
        K().attention_fp8(c.q, c.pages, c.scales, c.table, c.req, c.positions, out, *how, **kw)
    return out


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("mask", [dict(window=70), dict(window=901), dict(chunk=1000), dict(window=3000)])
def test_a_masked_first_tile_and_the_tiles_after_it(mask, dh, page):
    """The first tile's stage, with what lies before the window taken out of it, is filled again: large values stand there."""
    c = Case([1, 1, 1], [4010, 2999, 3333], 8, 2, dh, page)
    for r in range(3):
        p = c.held[r]
        lo = max(p - p % mask["chunk"] if "chunk" in mask else 0, p - mask["window"] + 1 if "window" in mask else 0)
        before = torch.arange(max(lo - 64, 0), lo)
        pages = c.table[r, before // page].long()
        c.pages.view(torch.uint8)[pages, :, :, before % page] = 0x7e  # 448
        c.scales[pages, :, :, before % page] = 127 + 60
    c.to_device()
    _serve(c, mask)
    want, tol = c.want(**mask)
    first = _call(c, mask)
    assert_close(first, want, tol)
    for _ in range(20):
        assert torch.equal(_call(c, mask), first)


@pytest.mark.parametrize("page", [16, 64])
def test_a_masked_first_tile_of_a_bfloat16_cache(page):
    c = Case([3, 2], [3001, 2600], 8, 2, 128, page, bits8=False).tree()
    for r in range(2):
        before = torch.arange(c.held[r] - 900 - 64, c.held[r] - 900)
        c.pages[c.table[r, before // page].long(), :, :, before % page] = math.inf
    c.to_device()
    _serve(c, dict(window=900))
    want, tol = c.want(window=900)
    first = _call(c, dict(window=900))
    assert_close(first, want, tol)
    for _ in range(20):
        assert torch.equal(_call(c, dict(window=900)), first)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_at_the_largest_scale_and_one_step_above(dtype):
    """448 * 2^60 is held, the next number of the type is not, nor is what lies just above the limit."""
    limit = 448 * 2.0 ** 60
    step = torch.finfo(dtype).eps * 2.0 ** 68  # (448 * 2^60 lies in [2^68, 2^69))
    tops = [limit, limit + step, limit + 2 * step, limit + 20 * step, limit - step, 2.0 * limit, -limit, -limit - step]
    c = Case([len(tops)], [2], 2, 2, 64, 16).to_device()
    k, v = torch.randn(len(tops), 2, 64, dtype=torch.float64), torch.randn(len(tops), 2, 64, dtype=torch.float64)
    for i, top in enumerate(tops):
        k[i, 0, 7], v[i, 1, 63] = top, -top
    k, v = k.to(dtype), v.to(dtype)
    assert float(k[1, 0, 7]) > limit and float(k[0, 0, 7]) == limit
    K().kv_store_fp8(k.cuda(), v.cuda(), c.pages, c.scales, c.table, c.req, c.places, c.status)
    _, want = hold(torch.stack([k, v], 1))
    assert torch.equal(c.scales[c.table[0, 0].long()][:, :, 2:2 + len(tops)].permute(2, 0, 1).cpu(), want)
    ko, vo = torch.empty_like(k, device="cuda"), torch.empty_like(v, device="cuda")
    K().kv_load_fp8(c.pages, c.scales, c.table, c.req, c.places, ko, vo, c.status)
    for got, x in ((ko, k), (vo, v)):
        x, _ = hold(x)
        assert torch.equal(torch.isnan(got).cpu(), torch.isnan(x)) and torch.equal(torch.nan_to_num(got.cpu().double()), torch.nan_to_num(x))


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 14, 2.0 ** -50])
def test_keys_that_were_never_written_count_as_zeros(form, n, size):
    """Scale byte 0, as the cache begins: a key of zeros, whose score is 0, and a value of zeros, in the sum like any other, whatever
    the scales of the values beside it."""
    c = Case([n], [300], 4, 2, 128, 16)
    c.rows[:, 1] *= size
    c.rows, scales = hold(c.rows)
    c.set_rows8(scales)
    for place in range(3, 300, 5):
        page, at = int(c.table[0, place // 16]), place % 16
        c.rows[page, :, :, at] = 0.0
        c.pages.view(torch.uint8)[page, :, :, at] = 0
        c.scales[page, :, :, at] = 0
    c.q *= 0.02  # scores close to each other: every key has its share of the sum
    c.to_device()
    assert_close(_call(c, items=c.items(n)), *c.want())


def _with_a_stranger_in_page_0(c):
    """Page 0 belongs to none of the case's requests, and holds values that would show in any output."""
    spare = next(p for p in range(1, c.P) if not (c.table == p).any())
    c.rows[spare] = c.rows[0]
    c.pages.view(torch.uint8)[spare] = c.pages.view(torch.uint8)[0]
    c.table[c.table == 0] = spare
    c.pages[0] = torch.full_like(c.pages[0], 300.0 if c.bits8 else 5e4)
    if c.bits8:
        c.scales[spare] = c.scales[0]
        c.scales[0] = 127 + 12
    return c


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("n, page, dh", [(1, 64, 128), (2, 16, 64), (40, 64, 64), (40, 16, 128), (90, 48, 128), (3, 24, 128), (40, 7, 64)])
@pytest.mark.parametrize("what", ["none", "too high"])
def test_a_missing_page_counts_as_keys_of_zeros(form, what, n, page, dh, bits8):
    """A request whose table names no page for some of its keys: the status says so, zeros stand in for them in every kernel, and no
    other request's rows enter its output."""
    c = _with_a_stranger_in_page_0(Case([n, n], [700, 333], 4, 2, dh, page, bits8=bits8).tree())
    for entry in (0, 300 // page, 640 // page):
        c.rows[int(c.table[0, entry])] = 0.0
    _serve(c)
    want, tol = c.want()
    for entry in (0, 300 // page, 640 // page):
        c.table[0, entry] = -1 if what == "none" else c.P + entry
    c.to_device()
    assert_close(_call(c), want, tol)
    assert int(c.status) == 1
    if bits8:
        c.masks = None
        c.positions = c.places.clone()
        c.status.zero_()
        table, c.table = c.table, c.table.clamp(0, c.P - 1)
        for entry in (0, 300 // page, 640 // page):  # (the oracle reads them as zeros: from a page of its own)
            c.table[0, entry] = 0
        c.rows[0] = 0.0
        _serve(c, items=c.items(n))
        want, tol = c.want()
        c.table = table
        assert_close(_call(c, items=c.items(n)), want, tol)
        assert int(c.status) == 1


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("n, page", [(1, 64), (3, 16), (60, 32)])
def test_pages_given_back_behind_a_window_are_not_asked_for(form, n, page, bits8):
    c = _with_a_stranger_in_page_0(Case([n], [2000], 4, 2, 128, page, bits8=bits8).tree())
    _serve(c, dict(window=700))
    want, tol = c.want(window=700)
    c.table[0, :(2000 - 700 + 1) // page] = -1
    c.to_device()
    assert_close(_call(c, dict(window=700)), want, tol)
    assert int(c.status) == 0


@pytest.mark.parametrize("form", ["attention_rows", "attention_rows_tc", "attention_few"], indirect=True)
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("cut", [3, 14])
def test_ranges_of_a_few_items_of_a_step_are_joined_from_scratch_of_their_own(monkeypatch, form, bits8, cut):
    """Items that are far fewer than the step's tokens, in pieces of any order, some shorter than the call was sized for."""
    monkeypatch.setattr(K(), "attention_rows_plan", lambda *a: (12, 128))
    c = Case([14, 200, 9], [900, 0, 1500], 8, 2, 128, 64, bits8=bits8).tree().to_device()
    items = c.items(cut, lambda n: n != 200)
    items = (items[0].flip(0).contiguous(), *items[1:])
    assert items[1] * items[2] < c.N
    out = _call(c, items=items)
    ours = [i for i in range(c.N) if not 14 <= i < 214]
    assert_close(out, *c.want(), ours)
    assert (out[14:214] == 7).all() and int(c.status) == 0


def test_one_token_behind_a_long_context_beside_a_portion_takes_little_memory():
    """40 heads on 8 of 128, 30,000 keys: the ranges of one row, not of the portion's 2,048 others."""
    c = Case([2048, 1], [0, 30000], 40, 8, 128, 64).to_device()
    row = torch.tensor([2048], dtype=torch.int32, device="cuda")
    out = torch.full_like(c.q, 7.0)
    _call(c, out=out, rows=row)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    _call(c, out=out, rows=row)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= 64 << 20
    alone = Case([1], [30000], 40, 8, 128, 64).to_device()
    alone.pages, alone.scales, alone.P, alone.rows, alone.q = c.pages, c.scales, c.P, c.rows, c.q[2048:].contiguous()
    alone.table = c.table[1:].contiguous()
    got = _call(alone)
    assert torch.equal(got[0], out[2048]) and (out[:2048] == 7).all()
    assert_close(got, *alone.want())


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("n", [3, 60])
@pytest.mark.parametrize("steps", [[5.0, 5.0], [15.0, 15.5], [3.0, 14.0], [40.0, 5.5]])
def test_large_values_of_a_bfloat16_cache_are_averaged_not_lost(form, n, steps):
    """Values of 2^126, a quarter of what the type holds, behind scores that climb: an average of them is finite."""
    c = Case([n], [900], 4, 1, 128, 16, bits8=False, spread=0.0).tree()
    c.q[:] = c.q[0, 0]
    c.rows[:, 0] *= 0.02
    top = 0.0
    for place, step in zip((300, 700), steps):
        top += step
        page, at = int(c.table[0, place // 16]), place % 16
        c.rows[page, 0, 0, at] = c.q[0, 0].double() * (top / (c.scale * math.log2(math.e) * float((c.q[0, 0].double() ** 2).sum())))
    c.rows[:, 1] = c.rows[:, 1].sign() * 2.0 ** 126 * torch.where(c.rows[:, 1].abs() > 1, 1.0, 0.5)
    c.pages = c.rows.to(torch.bfloat16)
    c.rows = c.pages.double()
    c.to_device()
    out = _call(c)
    assert torch.isfinite(out).all()
    assert_close(out, *c.want())


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("top", [2.0 ** 10, 2.0 ** 13, 2.0 ** 16, 2.0 ** 20])
@pytest.mark.parametrize("n, Hq, dh", [(2, 4, 128), (40, 8, 64), (70, 4, 128)])
def test_queries_with_one_entry_far_above_the_others(form, top, n, Hq, dh):
    """The large entry meets keys of zero: the scores are those of the small ones.  What the operands lose of an entry: nothing down
    to 2^-13 of the row's largest and 2^-21 of that below it (two 8-bit parts), 2^-32 of it (float16).  The values are +-1, so
    that a score's error d adds 2 d to an output's."""
    c = Case([n], [300], Hq, 2, dh, 16, spread=0.0)
    c.rows[:, 0, ..., 5] = 0.0
    c.rows[:, 1] = c.rows[:, 1].sign()
    c.rows, scales = hold(c.rows)
    c.set_rows8(scales)
    c.q[..., 5] = top
    c.to_device()
    items = c.items(n)
    out = _call(c, items=items)
    want, tol = c.want()
    part = 2.0 ** -21 if c.weights == 2.0 ** -8 else 2.0 ** -32
    size = float(c.rows[:, 0].abs().sum(-1).max()) * c.scale
    tol = tol + 2 * part * top * size
    assert_close(out, want, tol)


@pytest.mark.parametrize("n, held, Hq, Hkv, dh, page, mask", [
    ([20], [300], 4, 2, 64, 16, {}), ([5, 13], [700, 64], 8, 2, 128, 64, {}), ([8, 3, 8], [1000, 0, 333], 40, 8, 128, 64, {}), ([60], [900], 2, 2, 128, 48, dict(window=200)),
    ([16, 16], [2000, 100], 12, 3, 64, 32, dict(chunk=512)),
])
def test_few_items_of_17_to_64_rows_keep_float16s_digits(n, held, Hq, Hkv, dh, page, mask):
    """8-bit items that the rule sends to the few-rows kernel, held to its own bound, as portions and as trees."""
    c = Case(n, held, Hq, Hkv, dh, page).to_device()
    out = _call(c, mask, c.items(max(n)))
    assert c.weights == 2.0 ** -11 and 16 < max(n) * (Hq // Hkv) <= 64
    assert_close(out, *c.want(**mask))
    c = Case(n, held, Hq, Hkv, dh, page).tree().to_device()
    out = _call(c, mask)
    assert c.weights == 2.0 ** -11
    assert_close(out, *c.want(**mask))


def test_a_few_rows_of_a_step_on_two_streams_and_in_graphs():
    """Scratch that holds the served rows alone: calls at once on two streams, captured ones replayed with other queries, a row twice."""
    cases = [Case([1, 600, 1], [9000 + 700 * i, 0, 8000], 8, 2, 128, 64, seed=i).to_device() for i in range(2)]
    rows = torch.tensor([601, 0, 601], dtype=torch.int32, device="cuda")
    served, others = [0, 601], slice(1, 601)
    seen = K()._keys_seen(9702, 0, 0, 1)
    form = K().attention_rows_form(4, 64, True, seen, 6, True)
    assert form == "attention_few" and K().attention_rows_plan(form, 9702, 0, 0, 3, 1, 8, 2, 148)[0] > K().ROWS_CLUSTER

    def want(c):
        one = Case([1, 1], [c.held[0], c.held[2]], 8, 2, 128, 64)
        one.rows, one.table, one.q = c.rows, c.table[[0, 2]].contiguous(), c.q[served].contiguous()
        return one.want()

    sides = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for c, s in zip(cases, sides):
            with torch.cuda.stream(s):
                outs.append(_call(c, rows=rows))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert_close(out[served], *want(cases[i % 2]))
        assert (out[others] == 7).all()
    graphs = []
    for c in cases:
        out, g = torch.full_like(c.q, 7.0), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _call(c, rows=rows, out=out)
        graphs.append((g, out))
        c.q.mul_(0.5)
    for _ in range(2):
        for (g, _), c in zip(graphs, cases):
            g.replay()
            eager = _call(c, rows=rows)
    torch.cuda.synchronize()
    for (_, out), c in zip(graphs, cases):
        assert_close(out[served], *want(c))
        assert (out[others] == 7).all()
    assert torch.equal(eager, graphs[-1][1])
