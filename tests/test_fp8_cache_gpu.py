"""The 8-bit cache and the attention over it, and over drafted trees, against their definitions in 64 bits (fp8_helpers.py)."""

import math

import pytest
import torch

from .fp8_helpers import Case, assert_close, hold

pytestmark = pytest.mark.gpu


def K():
    from jax_llm_examples_b200.kernels import api

    return api


def cuda(t):
    return t.to("cuda")


# ------------------------------------------------------------------------------------------------ writing and reading back
def _rows(shape, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen) * torch.exp2(torch.randint(-20, 20, shape[:-1] + (1,), generator=gen).float())
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, held, Hkv, dh, page", [
    ([1], [0], 1, 64, 16), ([3, 1, 5], [7, 0, 61], 2, 128, 64), ([33, 2], [100, 14], 3, 24, 7), ([5], [2], 8, 256, 1), ([1500], [9], 4, 128, 48), ([9], [0], 5, 8, 4),
])
def test_rows_are_kept_as_the_format_says(dtype, n, held, Hkv, dh, page):
    c = Case(n, held, Hkv, Hkv, dh, page, seed=3).to_device()
    k, v = _rows((c.N, Hkv, dh), dtype, 1), _rows((c.N, Hkv, dh), dtype, 2)
    k[0, 0] = 0
    v[-1, -1] = 448.0  # the largest code, and the next scale's smallest top
    k[-1, -1, 0] = 448.0 * 1.5
    before = c.pages.view(torch.uint8).clone(), c.scales.clone()
    K().kv_store_fp8(cuda(k), cuda(v), c.pages, c.scales, c.table, c.req, c.places, c.status)
    want, bytes_ = hold(torch.stack([k, v], 1))
    page_of, at = c.table[c.req.long(), c.places.long() // page].long(), c.places.long() % page
    codes = c.pages.view(torch.uint8)[page_of, :, :, at].view(torch.float8_e4m3fn).cpu()
    got_bytes = c.scales[page_of, :, :, at].cpu()
    assert torch.equal(got_bytes, bytes_)
    assert torch.equal(codes.double() * torch.exp2(got_bytes.double() - 127)[..., None], want)
    for out_dtype in (torch.float32, torch.bfloat16):
        ko, vo = (torch.full((c.N, Hkv, dh), math.nan, dtype=out_dtype, device="cuda") for _ in range(2))
        K().kv_load_fp8(c.pages, c.scales, c.table, c.req, c.places, ko, vo, c.status)
        assert torch.equal(ko.cpu().double(), want[:, 0]) and torch.equal(vo.cpu().double(), want[:, 1])
    # every other row of the pool is as it was
    mine = torch.zeros((c.P, page), dtype=torch.bool, device="cuda")
    mine[page_of, at] = True
    keep = ~mine[:, None, None].expand(c.P, 2, Hkv, page)
    assert torch.equal(c.scales[keep], before[1][keep])
    assert torch.equal(c.pages.view(torch.uint8)[keep], before[0][keep])
    assert int(c.status) == 0


def test_ties_go_to_the_even_step_and_small_rows_keep_the_smallest_scale():
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    ties = ((codes[1:] + codes[:-1]) / 2)[None, None].repeat(1, 1, 1)
    x = torch.zeros(4, 1, 128)
    x[0, 0, :126], x[0, 0, 126] = ties[0, 0, :126], 448.0
    x[1] = x[0] * 2.0 ** -40
    x[2] = x[0] * 2.0 ** -64  # below the smallest scale's range: coarser, not lost
    x[3] = x[0] * 2.0 ** -120
    c = Case([4], [0], 1, 1, 128, 16).to_device()
    K().kv_store_fp8(cuda(x), cuda(-x), c.pages, c.scales, c.table, c.req, c.places, c.status)
    ko, vo = torch.empty(4, 1, 128, device="cuda"), torch.empty(4, 1, 128, device="cuda")
    K().kv_load_fp8(c.pages, c.scales, c.table, c.req, c.places, ko, vo, c.status)
    want, _ = hold(x)
    assert torch.equal(ko.cpu().double(), want) and torch.equal(vo.cpu().double(), -want)
    # half of e4m3's smallest step, 2^-9, at the smallest scale; 2^-4 of an entry above 2^-6 of the scale, as everywhere
    assert ((want[2:] - x[2:].double()).abs() <= (x[2:].double().abs() * 2.0 ** -4).clamp(min=2.0 ** -70)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan, 1e30])
def test_rows_that_8_bits_cannot_hold_read_back_as_nan(dtype, bad):
    c = Case([4], [3], 2, 2, 64, 16).to_device()
    k, v = _rows((4, 2, 64), dtype, 5), _rows((4, 2, 64), dtype, 6)
    k[1, 0, 63], v[2, 1, 0] = bad, bad
    K().kv_store_fp8(cuda(k), cuda(v), c.pages, c.scales, c.table, c.req, c.places, c.status)
    ko, vo = torch.empty_like(k, device="cuda"), torch.empty_like(v, device="cuda")
    K().kv_load_fp8(c.pages, c.scales, c.table, c.req, c.places, ko, vo, c.status)
    for got, x in ((ko, k), (vo, v)):
        want, _ = hold(x)
        assert torch.equal(torch.isnan(got).cpu(), torch.isnan(want)) and torch.equal(torch.nan_to_num(got.cpu().double()), torch.nan_to_num(want))


def test_views_that_do_not_start_on_16_bytes():
    c = Case([5], [3], 2, 2, 64, 16).to_device()
    k, v = _rows((5, 2, 64), torch.bfloat16, 5), _rows((5, 2, 64), torch.bfloat16, 6)
    off = lambda t: torch.cat([t.new_zeros(1), t.flatten()]).to("cuda")[1:].view(t.shape)  # noqa: E731
    K().kv_store_fp8(off(k), off(v), c.pages, c.scales, c.table, c.req, c.places, c.status)
    ko, vo = off(torch.zeros_like(k)), off(torch.zeros_like(v))
    K().kv_load_fp8(c.pages, c.scales, c.table, c.req, c.places, ko, vo, c.status)
    assert torch.equal(ko.cpu().double(), hold(k)[0]) and torch.equal(vo.cpu().double(), hold(v)[0])


@pytest.mark.parametrize("what", ["no page", "page too high", "place beyond the table", "negative place", "unknown request"])
def test_a_place_without_a_page_is_left_out(what):
    c = Case([3], [20], 2, 2, 64, 16)
    if what == "no page":
        c.table[0, 1] = -1  # places 20 .. 22
    elif what == "page too high":
        c.table[0, 1] = c.P
    elif what == "place beyond the table":
        c.places += 1000
    elif what == "negative place":
        c.places -= 1000
    else:
        c.req += 1
    c.to_device()
    before = c.pages.view(torch.uint8).clone(), c.scales.clone()
    x = torch.ones(3, 2, 64, device="cuda")
    K().kv_store_fp8(x, x, c.pages, c.scales, c.table, c.req, c.places, c.status)
    assert torch.equal(c.pages.view(torch.uint8), before[0]) and torch.equal(c.scales, before[1])
    assert int(c.status) == 1
    c.status.zero_()
    ko, vo = torch.ones_like(x), torch.ones_like(x)
    K().kv_load_fp8(c.pages, c.scales, c.table, c.req, c.places, ko, vo, c.status)
    assert int(c.status) == 1 and not ko.any() and not vo.any()


@pytest.mark.parametrize("n, held, Hq, Hkv, dh, splits, norm, rope", [
    ([1, 1, 1], [0, 5, 131000], 4, 2, 64, 5, True, True), ([7, 40], [3, 0], 5, 1, 128, 1, False, True), ([2], [1], 3, 3, 24, 2, True, False), ([1100], [0], 8, 2, 64, 1, True, True),
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_projected_rows_turn_are_normed_and_kept(dtype, n, held, Hq, Hkv, dh, splits, norm, rope):
    """q, and the rows before they are quantised, to 32-bit accuracy; what is kept is one rounding away from them (a value next
    to the middle of two steps may go either way)."""
    if splits > 1 and dtype == torch.bfloat16:
        dtype = torch.float32
    c = Case(n, [min(h, 500) for h in held], Hq, Hkv, dh, 16, seed=3).to_device()
    positions = torch.tensor([held[r] + j for r in range(len(n)) for j in range(n[r])], dtype=torch.int32)
    gen = torch.Generator().manual_seed(9)
    x = torch.randn((splits, c.N, (Hq + 2 * Hkv) * dh) if splits > 1 else (c.N, (Hq + 2 * Hkv) * dh), generator=gen).to(dtype)
    inv = 500000.0 ** (-torch.arange(0, dh, 2).float() / dh) if rope else None
    q = torch.empty((c.N, Hq, dh), dtype=torch.bfloat16, device="cuda")
    K().rope_kv_store_fp8(cuda(x), q, c.pages, c.scales, c.table, c.req, cuda(positions), None if inv is None else cuda(inv), norm, 1e-5, Hq, Hkv, dh,
                          c.status, splits, places=c.places)
    y = (x.double().sum(0) if splits > 1 else x.double()).view(c.N, Hq + 2 * Hkv, dh)
    size = y.abs().amax(-1, keepdim=True)
    qk, v = y[:, :Hq + Hkv].clone(), y[:, Hq + Hkv:]
    if rope:
        a = (positions.double()[:, None] * inv.double())[:, None]
        e, o = qk[..., 0::2].clone(), qk[..., 1::2].clone()
        qk[..., 0::2], qk[..., 1::2] = e * a.cos() - o * a.sin(), o * a.cos() + e * a.sin()
    # 32 bits: the partials' sums, a turn (four roundings, an angle good to 2^-21 or so), the norm's sum, root and division
    err = (8 + splits) * 2.0 ** -24 + (2.0 ** -20 if rope else 0)
    off = size * err
    if norm:
        r = torch.sqrt((qk * qk).mean(-1, keepdim=True) + 1e-5)
        qk, scale = qk / r, 1 / r
        off_qk = off[:, :Hq + Hkv] * scale + qk.abs() * (dh + 4) * 2.0 ** -24
    else:
        off_qk = off[:, :Hq + Hkv]
    got_q = q.cpu().double()
    assert ((got_q - qk[:, :Hq]).abs() <= 2.0 ** -8 * qk[:, :Hq].abs() + 1.01 * off_qk[:, :Hq]).all()
    ko, vo = (torch.empty((c.N, Hkv, dh), device="cuda") for _ in range(2))
    K().kv_load_fp8(c.pages, c.scales, c.table, c.req, c.places, ko, vo, c.status)
    for got, exact, slack in ((ko, qk[:, Hq:], off_qk[:, Hq:]), (vo, v, off[:, Hq + Hkv:])):
        # a kept value: 2^-4 of the entry, or half of the smallest step, 2^-10 of the row's power of two (which is at most top / 224)
        step = torch.maximum(exact.abs() * 2.0 ** -4, exact.abs().amax(-1, keepdim=True) / 224 * 2.0 ** -10)
        assert ((got.cpu().double() - exact).abs() <= step * (1 + 2.0 ** -20) + 1.1 * slack).all()
        same = (got.cpu().double() == hold(exact)[0]).double().mean()
        assert same >= 0.999, float(same)  # (entries within 2^-20 of a border, of 2^-4 between borders)
    assert int(c.status) == 0


# --------------------------------------------------------------------------------------------------------- attention
def _extras(Hq, sink, slopes, seed=11):
    gen = torch.Generator().manual_seed(seed)
    return (cuda(torch.randn(Hq, generator=gen)) if sink else None), (cuda(2.0 ** (-torch.rand(Hq, generator=gen) * 8)) if slopes else None)


def _attend(c, mask, items=None, rows=None, out=None, max_kv=None, **kw):
    out = torch.full_like(c.q, 7.0) if out is None else out
    lead = (c.q, c.pages, c.scales, c.table, c.req, c.positions, out, c.scale, mask.get("chunk", 0), mask.get("window", 0), mask.get("temper", 0.0),
            mask.get("floor", 1.0), c.status, max_kv or max(a + b for a, b in zip(c.n, c.held)))
    c.served(items[2] if items is not None else 1)
    if items is not None:
        kw |= dict(items=items[0], n_items=items[1], max_count=items[2])
    if rows is not None:
        kw |= dict(rows=rows, n_rows=rows.numel())
    K().attention_fp8(*lead, **kw)
    return out


SINGLE = [
    # held (one more is each request's own), heads, KV heads, head size, page, mask
    ([0], 5, 1, 128, 16, {}),
    ([62, 63, 64, 0], 10, 2, 128, 64, {}),
    ([1, 500, 2300], 40, 8, 128, 48, {}),
    ([777, 3], 16, 1, 64, 7, {}),
    ([900], 20, 1, 128, 64, {}),  # more heads than one group of rows
    ([400, 90], 70, 1, 64, 16, {}),  # ... than a block's
    ([5000], 8, 8, 128, 64, {}),
    ([4100, 129], 6, 3, 64, 128, dict(window=700)),
    ([1000, 511, 512], 8, 2, 128, 64, dict(chunk=512)),
    ([3000, 40], 8, 2, 128, 64, dict(chunk=512, window=100)),
    ([700, 0], 4, 2, 64, 1, dict(window=1)),
]


@pytest.mark.parametrize("held, Hq, Hkv, dh, page, mask", SINGLE)
def test_single_tokens(held, Hq, Hkv, dh, page, mask):
    c = Case([1] * len(held), held, Hq, Hkv, dh, page).to_device()
    assert_close(_attend(c, mask), *c.want(**mask))
    assert int(c.status) == 0


@pytest.mark.parametrize("sink, slopes, cap, temper", [(True, False, 0.0, 0.0), (False, True, 0.0, 0.0), (False, False, 2.0, 0.0), (False, False, 0.0, 0.3), (True, True, 3.0, 0.1)])
@pytest.mark.parametrize("dh", [64, 128])
def test_single_tokens_with_sinks_slopes_caps_and_temperature(dh, sink, slopes, cap, temper):
    c = Case([1, 1], [1200, 30], 12, 2, dh, 32).to_device()
    sink, slopes = _extras(12, sink, slopes)
    mask = dict(window=1000, temper=temper, floor=16.0)
    assert_close(_attend(c, mask, sink=sink, slopes=slopes, softcap=cap), *c.want(sink=sink, slopes=slopes, cap=cap, **mask))


PORTIONS = [
    ([2], [0], 2, 2, 128, 16, 128, {}),
    ([300, 17, 5], [0, 40, 1000], 10, 2, 128, 64, 128, {}),
    ([130, 64], [63, 1], 4, 1, 64, 48, 16, {}),
    ([200], [333], 8, 2, 64, 5, 64, dict(window=50)),
    ([260, 31], [100, 0], 5, 1, 128, 64, 128, dict(chunk=128)),
    ([90], [2000], 3, 3, 128, 64, 33, dict(chunk=1024, window=600)),
]


FORMS = ["rule", "attention_rows", "attention_rows_tc", "attention_few"]  # the kernel by the sizes, or the one named where it can


@pytest.fixture
def form(request, monkeypatch):
    rule = K().attention_rows_form
    if request.param == "attention_rows_tc":
        monkeypatch.setattr(K(), "attention_rows_form", lambda rows, page, aligned, *a: request.param if page % 16 == 0 and aligned else rule(rows, page, aligned))
    elif request.param != "rule":
        monkeypatch.setattr(K(), "attention_rows_form", lambda *a: request.param)


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("n, held, Hq, Hkv, dh, page, cut, mask", PORTIONS)
def test_portions(form, n, held, Hq, Hkv, dh, page, cut, mask):
    c = Case(n, held, Hq, Hkv, dh, page).to_device()
    assert_close(_attend(c, mask, c.items(cut)), *c.want(**mask))
    assert int(c.status) == 0


def test_portions_beside_single_tokens_write_their_own_rows_only():
    c = Case([40, 1, 3, 1], [10, 600, 0, 77], 8, 2, 128, 64).to_device()
    sink, slopes = _extras(8, True, True)
    out = _attend(c, {}, c.items(16, lambda n: n > 1), sink=sink, slopes=slopes, softcap=5.0)
    single = [40, 44]
    assert (out[single] == 7).all()
    want, tol = c.want(sink=sink, slopes=slopes, cap=5.0)
    others = [i for i in range(c.N) if i not in single]
    assert_close(out, want, tol, others)
    _attend(c, {}, rows=torch.tensor(single, dtype=torch.int32, device="cuda"), out=out, sink=sink, slopes=slopes, softcap=5.0)
    assert_close(out, want, tol, others)
    assert_close(out, *c.want(sink=sink, slopes=slopes, cap=5.0), single)


@pytest.mark.parametrize("planned", [1, 64, 5000, 100000])
def test_the_planned_length_bounds_nothing(planned):
    c = Case([1, 1], [1500, 20], 8, 2, 128, 64).to_device()
    assert_close(_attend(c, {}, max_kv=planned), *c.want())


@pytest.mark.parametrize("form", FORMS, indirect=True)
def test_rows_of_very_different_scales(form):
    """Keys and values whose rows' scales lie tens of binades apart: a token that sees only small values keeps their digits."""
    c = Case([1, 1, 64], [300, 4, 0], 4, 2, 128, 16, spread=12.0)
    c.rows[..., 0, :, :, :] /= c.rows[..., 0, :, :, :].abs().amax(-1, keepdim=True).clamp(min=1e-30)  # keys of one size: scores stay moderate
    c.rows, s = hold(c.rows)
    c.set_rows8(s)
    c.to_device()
    out = _attend(c, {}, rows=torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    assert_close(out, *c.want(), [0, 1])
    _attend(c, {}, c.items(64, lambda n: n > 1), out=out)
    assert_close(out, *c.want(), slice(2, None))


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("places", [[700], [130, 500, 890], [3], [905]])
def test_scores_that_leap(form, bits8, places):
    """Keys whose scores swamp all before them, tiles apart, and a value for each to tell them by."""
    c = Case([30], [900], 8, 2, 128, 16, bits8=False).tree()
    for i, place in enumerate(places):
        page, at = int(c.table[0, place // 16]), place % 16
        c.rows[page, 0, :, at] *= 64.0 * 4.0 ** i
        c.rows[page, 1, :, at] = 96.0 + 32 * i  # (held exactly in either type)
    if bits8:
        c.rows, scales = hold(c.rows)
        c.set_rows8(scales)
        c.bits8 = True
    else:
        c.pages = c.rows.to(torch.bfloat16)
    c.to_device()
    out = _tree(c, {})
    want, tol = c.want()
    assert ((want > 95).all(-1) & (want < 161).all(-1)).any()
    assert_close(out, want, tol)


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("n", [3, 30, 70])
@pytest.mark.parametrize("steps", [[5.0, 5.0, 5.0], [12.0, 12.0, 15.0], [17.0, 5.0, 15.5], [-40.0, 15.0, 30.0]])
def test_scores_that_climb(form, bits8, n, steps):
    """The largest score of every row climbs by these powers of two, tiles apart: within what a reference may be outgrown by, and beyond."""
    c = Case([n], [900], 4, 1, 128, 16, bits8=False, spread=0.0).tree()
    c.q[:] = c.q[0, 0]
    c.rows[:, 0] *= 0.25
    top = 0.0
    for place, step in zip((150, 420, 800), steps):
        top += step
        page, at = int(c.table[0, place // 16]), place % 16
        c.rows[page, 0, 0, at] = c.q[0, 0].double() * (top / (c.scale * math.log2(math.e) * float((c.q[0, 0].double() ** 2).sum())))
    c.rows = c.rows.to(torch.bfloat16).double()
    if bits8:
        c.rows, scales = hold(c.rows)
        c.set_rows8(scales)
        c.bits8 = True
    else:
        c.pages = c.rows.to(torch.bfloat16)
    c.to_device()
    assert_close(_tree(c, {}), *c.want())


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("n", [8, 100])
def test_nan_rows_reach_those_that_see_them_and_no_other(form, n):
    c = Case([n], [50], 4, 2, 128, 16)
    at_token = n * 3 // 8
    place = 50 + at_token  # a key and a value, of different heads, in the middle of the portion
    page, at = int(c.table[0, place // 16]), place % 16
    c.rows[page, 0, 0, at], c.rows[page, 1, 1, at] = math.nan, math.nan
    c.scales[page, 0, 0, at], c.scales[page, 1, 1, at] = 255, 255
    c.to_device()
    out = _attend(c, {}, c.items(128))
    want, tol = c.want()
    assert torch.isnan(want[at_token:]).all() and not torch.isnan(want[:at_token]).any()
    assert_close(out, want, tol)


@pytest.mark.parametrize("n, dh, page", [(5, 64, 64), (2, 128, 16), (40, 128, 64), (40, 64, 16), (3, 128, 5)])
def test_stale_rows_behind_a_request_stay_out(n, dh, page):
    c = Case([n], [60], 4, 2, dh, page).to_device()
    c.pages.view(torch.uint8).masked_fill_(~_live(c)[..., None], 0x7f)  # NaN codes, NaN scales
    c.scales.masked_fill_(~_live(c), 255)
    assert_close(_attend(c, {}, c.items(n)), *c.want())


def _live(c):
    """[P, 2, Hkv, page]: the cache's rows that belong to a request."""
    live = torch.zeros((c.P, c.page), dtype=torch.bool, device="cuda")
    for r, (a, b) in enumerate(zip(c.n, c.held)):
        place = torch.arange(a + b, device="cuda")
        live[c.table[r, place // c.page].long(), place % c.page] = True
    return live[:, None, None].expand(c.P, 2, c.Hkv, c.page)


def test_a_bad_page_raises_the_status_and_no_more():
    c = Case([1, 1], [100, 100], 4, 2, 64, 16)
    c.table[0, 2], c.table[0, 3] = c.P + 5, -1
    c.to_device()
    out = _attend(c, {})
    assert int(c.status) == 1
    good = Case([1, 1], [100, 100], 4, 2, 64, 16).to_device()
    assert torch.equal(out[1], _attend(good, {})[1])


# ------------------------------------------------------------------------------------------------------ drafted trees
def _tree(c, mask, items=None, out=None, max_kv=None, **kw):
    out = torch.full_like(c.q, 7.0) if out is None else out
    items = items or c.items(max(c.n))
    c.served(items[2])
    K().attention_tree(c.q, c.pages, c.table, c.req, c.positions, c.cu_q, c.q_start, c.masks, out, c.scale, mask.get("chunk", 0), mask.get("window", 0),
                       mask.get("temper", 0.0), mask.get("floor", 1.0), c.status, max_kv or max(a + b for a, b in zip(c.n, c.held)), *items, scales=c.scales, **kw)
    return out


TREES = [
    ([1], [0], 4, 2, 128, 16, {}),
    ([7, 1, 13], [100, 0, 63], 10, 2, 128, 64, {}),
    ([32, 33], [1200, 64], 5, 1, 128, 48, {}),
    ([64, 20], [300, 2500], 12, 4, 64, 16, {}),
    ([100], [700], 8, 1, 128, 64, {}),
    ([31, 65], [128, 500], 40, 8, 128, 64, dict(window=200)),
    ([24], [510], 6, 2, 64, 7, dict(chunk=512)),
    ([40, 3], [1000, 2000], 4, 4, 128, 128, dict(chunk=1024, window=300, temper=0.2, floor=64.0)),
]


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("n, held, Hq, Hkv, dh, page, mask", TREES)
def test_trees(form, n, held, Hq, Hkv, dh, page, mask, bits8):
    c = Case(n, held, Hq, Hkv, dh, page, bits8=bits8).tree().to_device()
    assert_close(_tree(c, mask), *c.want(**mask))
    assert int(c.status) == 0


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("cut", [4, 7, 50])
def test_trees_with_sinks_slopes_and_caps_in_pieces(form, bits8, cut):
    c = Case([50, 9], [900, 64], 8, 2, 128, 64, bits8=bits8).tree().to_device()
    sink, slopes = _extras(8, True, True)
    out = _tree(c, {}, c.items(cut), sink=sink, slopes=slopes, softcap=4.0)  # a tree cut into several items
    assert_close(out, *c.want(sink=sink, slopes=slopes, cap=4.0))


@pytest.mark.parametrize("bits8", [False, True])
def test_a_chain_is_a_portion(bits8):
    c = Case([20], [300], 4, 2, 64, 16, bits8=bits8).tree(parents=[list(range(-1, 19))]).to_device()
    out = _tree(c, {})
    assert_close(out, *c.want())
    if bits8:
        c.masks = None
        assert_close(_attend(c, {}, c.items(20)), *c.want())


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("sink", [False, True])
def test_tokens_whose_mask_leaves_nothing_are_zero(form, bits8, sink):
    c = Case([6, 40], [0, 0], 4, 2, 128, 16, bits8=bits8).tree()
    c.masks[2] = 0
    c.masks[6 + 33:] = 0
    c.to_device()
    sink, _ = _extras(4, sink, False)
    out = _tree(c, {}, sink=sink)
    assert_close(out, *c.want(sink=sink))
    assert not out[2].any() and not out[6 + 33:].any()


@pytest.mark.parametrize("bits8", [False, True])
def test_bits_beyond_a_requests_tokens_mean_nothing(bits8):
    c = Case([5, 3], [40, 100], 4, 2, 64, 16, bits8=bits8).tree()
    want = c.want()
    c.masks[5:] |= -(1 << 3)
    c.masks[:5] |= -(1 << 5)
    c.to_device()
    assert_close(_tree(c, {}), *want)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("n, Hq", [(7, 4), (12, 4), (60, 8), (30, 16)])
@pytest.mark.parametrize("form", FORMS, indirect=True)
def test_infinite_and_nan_rows_of_a_bfloat16_cache_reach_those_that_see_them(form, n, Hq, bad):
    """Values that are not finite in a drafted token's row, and behind the last: only its descendants get them, in those entries."""
    c = Case([n, 2], [70, 5], Hq, 2, 128, 16, bits8=False).tree()
    place = 70 + 3
    page, at = int(c.table[0, place // 16]), place % 16
    c.rows[page, 1, 0, at, 5], c.rows[page, 1, 1, at, 127] = bad, bad
    c.pages = c.rows.to(torch.bfloat16)
    c.to_device()
    c.pages.masked_fill_(~_live(c)[..., None], bad)
    out = _tree(c, {}).cpu().double()
    want, tol = c.want()
    sees = [bool(int(c.masks[i, 0].cpu()) >> 3 & 1) for i in range(n)] + [False, False]
    hit = torch.zeros_like(want, dtype=torch.bool)
    hit[sees, :Hq // 2, 5] = True
    hit[sees, Hq // 2:, 127] = True
    assert any(sees) and not all(sees)
    if math.isnan(bad):
        assert torch.isnan(out[hit]).all()
    else:
        assert (out[hit] == bad).all()
    assert_close(torch.where(hit, torch.zeros_like(out), out), torch.where(hit, torch.zeros_like(want), want), tol.nan_to_num(0.0, 0.0))


def test_nan_keys_of_a_bfloat16_cache_reach_those_that_see_them():
    c = Case([12], [70], 4, 2, 64, 16, bits8=False).tree()
    place = 70 + 2
    c.rows[int(c.table[0, place // 16]), 0, 0, place % 16, 9] = math.nan
    c.pages = c.rows.to(torch.bfloat16)
    c.to_device()
    assert_close(_tree(c, {}, softcap=3.0), *c.want(cap=3.0))


# --------------------------------------------------------------------------------- streams, graphs, refusals on the GPU
def test_two_streams_at_once_and_a_captured_call():
    a, b = (Case([1, 1], [3000, 100 + i], 8, 2, 128, 64, seed=i).to_device() for i in range(2))
    sides = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for c, s in zip((a, b), sides):
            with torch.cuda.stream(s):
                outs.append(_attend(c, {}))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert_close(out, *(a, b)[i % 2].want())
    graphs = []
    for c in (a, b):
        out = torch.zeros_like(c.q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _attend(c, {}, out=out)
        graphs.append((g, out))
    for c in (a, b):
        c.q.mul_(0.5)
    for g, _ in graphs + graphs:
        g.replay()
    torch.cuda.synchronize()
    for (_, out), c in zip(graphs, (a, b)):
        assert_close(out, *c.want())


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 12])
@pytest.mark.parametrize("row_block", [128, 256])
@pytest.mark.parametrize("n, held, dh, mask", [
    (60, 700, 128, {}),  # 300 rows: 256 and 44, or 128, 128 and 44
    (26, 100, 64, {}),  # 130 rows on one tile of keys and on two
    (51, 1000, 64, dict(window=300)),
    (52, 129, 128, dict(chunk=128)),  # 260 rows
])
def test_rows_of_a_block_and_ranges(monkeypatch, n, held, dh, mask, row_block, splits, bits8):
    """Either number of rows, with fewer tiles of keys than ranges and with ranges of one tile, two and more."""
    monkeypatch.setattr(K(), "attention_rows_plan", lambda *a: (splits, row_block))
    c = Case([n, 3], [held, 5], 5, 1, dh, 64, bits8=bits8).tree().to_device()
    assert_close(_tree(c, mask), *c.want(**mask))
    if bits8:
        c = Case([n, 3], [held, 5], 5, 1, dh, 48).to_device()
        sink, _ = _extras(5, True, False)
        assert_close(_attend(c, mask, c.items(n), sink=sink), *c.want(sink=sink, **mask))
    assert int(c.status) == 0


@pytest.mark.parametrize("cut", [1, 40])
@pytest.mark.parametrize("bits8", [False, True])
def test_a_cache_past_31_bits(bits8, cut):
    """Pages that begin more than 2^31 bytes (and, in 16 bits, numbers) behind the cache's start."""
    c = Case([40], [300], 8, 1, 128, 64, bits8=bits8).tree().to_device()
    pool = torch.empty((2 ** 31 // (2 * 64 * 128) + 100 + c.P, *c.pages.shape[1:]), dtype=c.pages.dtype, device="cuda")
    at = pool.shape[0] - c.P
    pool.view(torch.uint8)[at:] = c.pages.view(torch.uint8)
    if bits8:
        scales = torch.zeros((pool.shape[0], *c.scales.shape[1:]), dtype=torch.uint8, device="cuda")
        scales[at:] = c.scales
        c.scales = scales
    c.pages = pool
    c.table = torch.where(c.table >= 0, c.table + at, c.table)
    table, c.table = c.table, c.table - at  # (want() reads the small pool)
    want, tol = c.want()
    c.table = table
    c.served(cut)
    assert_close(_tree(c, {}, c.items(cut)), want, tol)
    if bits8:
        x = torch.randn(40, 1, 128, device="cuda")
        ko, vo = torch.empty_like(x), torch.empty_like(x)
        K().kv_store_fp8(x, -x, pool, c.scales, c.table, c.req, c.places, c.status)
        K().kv_load_fp8(pool, c.scales, c.table, c.req, c.places, ko, vo, c.status)
        assert torch.equal(ko.cpu().double(), hold(x.cpu())[0]) and torch.equal(vo, -ko)
    assert int(c.status) == 0


def test_ranges_of_many_rows_on_two_streams_and_in_two_graphs():
    """The calls whose ranges are joined through scratch: at once on two streams, and captured twice and replayed in turn with an eager call."""
    cases = [Case([60], [3000 + 64 * i], 10, 2, 128, 64, seed=i, bits8=i > 0).tree(seed=i).to_device() for i in range(2)]
    cases.append(Case([1], [9000], 8, 2, 128, 64).to_device())  # single tokens in more ranges than a cluster joins
    items = {id(c): c.items(max(c.n)) for c in cases}  # (made before the captures)
    call = lambda c, out: _tree(c, {}, items[id(c)], out=out) if c.masks is not None else _attend(c, {}, out=out)  # noqa: E731
    for c in cases:
        form = K().attention_rows_form(max(c.n) * (c.Hq // c.Hkv), c.page, True)
        joined = K().ROWS_CLUSTER if form == "attention_few" else 1
        sms = torch.cuda.get_device_properties(0).multi_processor_count
        assert K().attention_rows_plan(form, c.held[0] + c.n[0], 0, 0, 1, max(c.n), c.Hq, c.Hkv, sms)[0] > joined
    want = [c.want() for c in cases]
    sides = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for c, s in zip(cases, sides):
            with torch.cuda.stream(s):
                outs.append(call(c, torch.zeros_like(c.q)))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert_close(out, *want[i % 3])
    graphs = []
    for c in cases + cases:
        out, g = torch.zeros_like(c.q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(c, out)
        graphs.append((g, out))
    for _ in range(2):
        for g, out in graphs:
            out.zero_()
            g.replay()
            eager = call(cases[0], torch.zeros_like(cases[0].q))
    torch.cuda.synchronize()
    assert_close(eager, *want[0])
    for i, (_, out) in enumerate(graphs):
        assert_close(out, *want[i % 3])


@pytest.mark.parametrize("n", [1, 9, 40])
def test_scales_that_do_not_start_on_16_bytes(n):
    c = Case([n], [200], 8, 2, 128, 64).to_device()
    c.scales = torch.cat([c.scales.new_zeros(1), c.scales.flatten()])[1:].view(c.scales.shape)
    assert c.scales.data_ptr() % 16
    c.weights = 2.0 ** -11
    out = torch.full_like(c.q, 7.0)
    items = c.items(n)
    K().attention_fp8(c.q, c.pages, c.scales, c.table, c.req, c.positions, out, c.scale, 0, 0, 0.0, 1.0, c.status, 200 + n, items=items[0], n_items=items[1],
                      max_count=items[2])
    assert_close(out, *c.want())


def test_steps_of_no_tokens_and_rows_asked_for_twice():
    c = Case([3, 1], [20, 30], 4, 2, 64, 16).to_device()
    none = c.q[:0]
    K().attention_fp8(none, c.pages, c.scales, c.table, c.req[:0], c.positions[:0], torch.empty_like(none), c.scale, 0, 0, 0.0, 1.0, c.status, 1)
    k = torch.empty(0, 2, 64, device="cuda")
    K().kv_store_fp8(k, k, c.pages, c.scales, c.table, c.req[:0], c.places[:0], c.status)
    K().kv_load_fp8(c.pages, c.scales, c.table, c.req[:0], c.places[:0], k, torch.empty_like(k), c.status)
    out = _attend(c, {}, (torch.zeros((1, 2), dtype=torch.int32, device="cuda"), 0, 1))
    assert (out == 7).all()
    _attend(c, {}, (torch.tensor([[0, 3], [1, 2], [0, 0]], dtype=torch.int32, device="cuda"), 3, 3), out=out)  # rows 1 and 2 twice; an item of none
    _attend(c, {}, rows=torch.tensor([3, 3, 3], dtype=torch.int32, device="cuda"), out=out)
    assert_close(out, *c.want())
    assert int(c.status) == 0


def test_a_description_that_points_outside_the_step_is_refused_by_the_kernel():
    c = Case([4], [20], 4, 2, 64, 16).tree().to_device()
    for items in ([[2, 3]], [[-1, 2]], [[0, 9]]):
        c.status.zero_()
        _tree(c, {}, (torch.tensor(items, dtype=torch.int32, device="cuda"), 1, 9))
        assert int(c.status) == 1
    for most in (1, 3):  # an item of more tokens than the call was sized for
        c.status.zero_()
        out = _tree(c, {}, (torch.tensor([[0, 4]], dtype=torch.int32, device="cuda"), 1, most))
        assert int(c.status) == 1 and (out == 7).all()
    c.status.zero_()
    out = _attend(c, {}, rows=torch.tensor([1, 77], dtype=torch.int32, device="cuda"))
    assert int(c.status) == 1 and (out[0] == 7).all() and not (out[1] == 7).all()


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("n", [2, 40])
@pytest.mark.parametrize("far", [10 ** 4, 2 ** 31 - 1])
def test_positions_that_the_table_cannot_hold_raise_the_status(form, n, far):
    c = Case([n, n], [20, 30], 8, 2, 64, 16).to_device()
    c.positions[n - 1] = far
    out = _attend(c, {}, c.items(n))
    assert int(c.status) == 1
    c.positions[n - 1] = 20 + n - 1
    assert_close(out, *c.want(), slice(n, None))  # the other request's rows
    c.status.zero_()
    c.positions[:n] = -5000  # before the first key: nothing is seen
    out = _attend(c, dict(chunk=512), c.items(n))
    assert not out[:n].any() and int(c.status) == 0


@pytest.mark.parametrize("n", [2, 40])
@pytest.mark.parametrize("far", [10 ** 4, 2 ** 31 - 1])
def test_trees_that_the_table_cannot_hold_raise_the_status(n, far):
    c = Case([n, n], [20, 30], 8, 2, 64, 16).tree().to_device()
    c.q_start[0] = far
    out = _tree(c, {})
    assert int(c.status) == 1
    c.q_start[0] = 20
    assert_close(out, *c.want(), slice(n, None))


def test_head_sizes_without_a_kernel_are_refused():
    c = Case([1], [20], 4, 2, 32, 16).to_device()
    with pytest.raises(K().KernelError, match="not supported"):
        _attend(c, {})
    assert not K().attention_rows_supported(torch.bfloat16, 4, 2, 32) and K().attention_rows_supported(torch.bfloat16, 4, 2, 64)
    assert not K().attention_rows_supported(torch.float32, 4, 2, 64)


def test_a_step_written_read_and_extended_by_a_tree():
    """As they are used together: a prompt and then a drafted tree are written in 8 bits and attended, the tree behind the prompt."""
    Hq, Hkv, dh, T, D = 8, 2, 128, 150, 21
    c = Case([D], [T], Hq, Hkv, dh, 64).tree().to_device()
    gen = torch.Generator(device="cuda").manual_seed(4)
    inv = 10000.0 ** (-torch.arange(0, dh, 2, device="cuda").float() / dh)
    for n, first, positions, places in ((T, 0, torch.arange(T), torch.arange(T)), (D, T, c.positions.cpu(), T + torch.arange(D))):
        qkv = torch.randn((n, (Hq + 2 * Hkv) * dh), generator=gen, device="cuda").to(torch.bfloat16)
        q = torch.empty((n, Hq, dh), dtype=torch.bfloat16, device="cuda")
        req = torch.zeros(n, dtype=torch.int32, device="cuda")
        positions, places = cuda(positions.to(torch.int32)), cuda(places.to(torch.int32))
        K().rope_kv_store_fp8(qkv, q, c.pages, c.scales, c.table, req, positions, inv, True, 1e-6, Hq, Hkv, dh, c.status, places=places)
        step = Case([n], [first], Hq, Hkv, dh, 64)
        step.q, step.positions, step.table, step.page, step.masks = q, positions, c.table, 64, c.masks if first else None
        step.rows = (c.pages.float() * torch.exp2(c.scales.float() - 127)[..., None]).double().cpu()
        out = torch.empty_like(q)
        step.served(n if first else 100)
        if first:
            c.q = q
            _tree(c, {}, out=out)
        else:
            K().attention_fp8(q, c.pages, c.scales, c.table, req, positions, out, c.scale, 0, 0, 0.0, 1.0, c.status, n,
                              items=torch.tensor([[0, 100], [100, 50]], dtype=torch.int32, device="cuda"), n_items=2, max_count=100)
        assert_close(out, *step.want())
    assert int(c.status) == 0
