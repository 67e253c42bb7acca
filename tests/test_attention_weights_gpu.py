"""The weights that cached keys receive, from single tokens, last tokens of prompts and whole portions, against the definition in 64 bits."""

import math

import pytest
import torch

from .budget_helpers import received
from .fp8_helpers import Case, assert_close, two_to

pytestmark = pytest.mark.gpu


def K():
    from jax_llm_examples_b200.kernels import api

    return api


def run(c, width=None, add=None, out=None, cu_q=None, max_kv=None, max_count=None, status=None, chunk=0, window=0, temper=0.0, floor=1.0, sink=None, slopes=None,
        cap=0.0):
    width = width or max(a + b for a, b in zip(c.n, c.held))
    out = torch.full((len(c.n), c.Hkv, width), math.nan, device="cuda") if out is None else out
    K().attention_weights(c.q, c.pages, c.table, c.cu_q if cu_q is None else cu_q, c.positions, out, c.scale, chunk, window, temper, floor,
                          c.status if status is None else status, max_kv or max(a + b for a, b in zip(c.n, c.held)), max_count or max(c.n), scales=c.scales,
                          sink=sink, slopes=slopes, softcap=cap, add=add)
    return out


# (tokens of each request, keys before them, query heads, KV heads, head size, page)
STEPS = {
    "one of one": ([1], [0], 8, 8, 128, 16),
    "one": ([1], [699], 40, 8, 128, 64),
    "ragged": ([1, 1, 1, 1, 1], [0, 15, 16, 300, 1023], 40, 8, 128, 64),
    "small heads": ([1, 1, 1], [64, 517, 90], 16, 4, 64, 48),
    "group of 16": ([1, 1], [333, 12], 32, 2, 128, 16),
    "no group": ([1, 1], [250, 77], 6, 6, 64, 7),
    "three tokens": ([3, 3, 1], [100, 513, 31], 16, 4, 128, 32),
    "long": ([1], [9000], 8, 2, 128, 64),
    "some without": ([1, 0, 2, 0], [5, 40, 700, 0], 8, 4, 64, 16),
}


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("step", STEPS)
def test_few_rows(step, bits8):
    n, held, Hq, Hkv, dh, page = STEPS[step]
    c = Case(n, held, Hq, Hkv, dh, page, seed=len(step), bits8=bits8).to_device()
    want, tol = received(c)
    assert_close(run(c), want, tol)
    assert int(c.status) == 0


MASKS = {
    "chunk": dict(chunk=128), "window": dict(window=77), "both": dict(chunk=256, window=100), "temperature": dict(temper=0.1, floor=64.0), "cap": dict(cap=5.0),
    "sink": dict(sink=True), "slopes": dict(slopes=True), "all": dict(window=200, temper=0.2, floor=32.0, cap=20.0, sink=True, slopes=True),
}


def _masks(c, mask):
    gen = torch.Generator().manual_seed(3)
    a = dict(MASKS[mask])
    if a.get("sink"):
        a["sink"] = torch.randn(c.Hq, generator=gen).cuda()
    if a.get("slopes"):
        a["slopes"] = (0.1 * torch.rand(c.Hq, generator=gen)).cuda()
    return a


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("mask", MASKS)
def test_masks_and_scores_of_few_rows(mask, bits8):
    c = Case([1, 2, 1], [400, 300, 20], 16, 4, 64, 16, seed=5, bits8=bits8).to_device()
    a = _masks(c, mask)
    want, tol = received(c, **a)
    assert_close(run(c, **a), want, tol)


@pytest.mark.parametrize("n", [[1, 1], [2, 1]])
def test_adds_to_what_is_there_and_writes_every_place(n):
    c = Case(n, [130, 57], 8, 4, 128, 16, bits8=False).to_device()
    width = 200
    add = torch.rand((2, 4, width), generator=torch.Generator().manual_seed(1)).cuda()
    want, tol = received(c, add=add, width=width)
    assert_close(run(c, width=width, add=add), want, tol)
    assert torch.equal(run(c, width=width, add=add)[:, :, 150:], add[:, :, 150:])
    assert_close(run(c, width=width), *received(c, width=width))
    there = add.clone()
    run(c, width=width, add=there, out=there)
    assert_close(there, want, tol)


def test_a_row_that_sees_nothing_gives_nothing():
    c = Case([1, 1], [50, 60], 8, 4, 64, 16, bits8=False)
    c.positions[0] = -1
    c.to_device()
    want, tol = received(c)
    assert float(want[0].sum()) == 0
    for sink in (None, torch.zeros(8, device="cuda")):
        got = run(c, sink=sink)
        assert float(got[0].abs().sum()) == 0 and not bool(got.isnan().any())
    assert_close(run(c), want, tol)


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("n", [[1, 1], [40, 3]])
def test_what_is_masked_may_be_anything(n, bits8):
    """Keys behind the last one and before the window hold infinities and NaN."""
    c = Case(n, [200, 100], 8, 4, 128, 16, seed=2, bits8=bits8)
    window = 60
    want, tol = received(c, window=window)
    for r in range(2):
        for place in list(range(c.held[r] - window)) + list(range(c.held[r] + c.n[r], -(-(c.held[r] + c.n[r]) // 16) * 16)):
            page = int(c.table[r, place // 16])
            if bits8:
                c.scales[page, :, :, place % 16] = 255
            else:
                c.pages[page, :, :, place % 16] = math.nan if place % 2 else math.inf
    c.to_device()
    assert_close(run(c, window=window), want, tol)


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("n", [[1, 1], [20, 2]])
def test_a_visible_nan_spoils_its_rows_only(n, bits8):
    c = Case(n, [90, 100], 8, 4, 64, 16, seed=2, bits8=bits8)
    page, at = int(c.table[1, 2]), 5
    if bits8:
        c.scales[page, 0, 1, at] = 255
    else:
        c.pages[page, 0, 1, at] = math.nan
    c.to_device()
    got = run(c)
    assert bool(got[1, 1, :c.held[1] + 1].isnan().all())
    bad = got.isnan()
    bad[1, 1] = False
    assert not bool(bad.any())


@pytest.mark.parametrize("n", [[1, 1], [30, 1]])
def test_missing_pages_are_zeros_and_raise_the_status(n):
    c = Case(n, [100, 100], 8, 4, 128, 16, bits8=False)
    c.rows[c.table[0, 1].long()] = 0
    want, tol = received(c)
    c.table[0, 1] = 10000
    c.to_device()
    assert_close(run(c), want, tol)
    assert int(c.status) == 1
    c.status.zero_()
    # beyond what any row sees nothing is looked at
    c.table[0, -1] = -5
    c.table[0, 1] = 3
    run(c)
    assert int(c.status) == 0


@pytest.mark.parametrize("n", [[1, 1], [30, 30]])
def test_more_than_the_call_was_sized_for_gives_nothing(n):
    c = Case(n, [2000, 30], 8, 4, 128, 16, bits8=False).to_device()
    want, tol = received(c)
    add = torch.rand_like(want, dtype=torch.float32).cuda()
    for change in (dict(max_kv=100), dict(cu_q=torch.tensor([0, c.N + 1, c.N], dtype=torch.int32).cuda())):
        c.status.zero_()
        got = run(c, add=add, **change)
        assert torch.equal(got[0], add[0]) and int(c.status) == 1
    c.status.zero_()
    got = run(c, width=100)
    assert float(got[0].abs().sum()) == 0 and int(c.status) == 1
    assert_close(got[1], want[1, :, :100], tol[1, :, :100])


@pytest.mark.parametrize("bits8", [False, True])
def test_ranges_too_long_for_shared_memory(monkeypatch, bits8):
    """Their scores go through scratch: at the size where they do, and as if shared memory were small."""
    assert not K().attention_weights_plan(500000, 1, 8, 148)[2]
    plan = K().attention_weights_plan
    monkeypatch.setattr(K(), "attention_weights_plan", lambda *a: (*plan(*a)[:2], False))
    c = Case([1, 2], [9000, 333], 8, 2, 64, 64, bits8=bits8).to_device()
    want, tol = received(c)
    assert_close(run(c), want, tol)


@pytest.mark.parametrize("n", [[1, 1, 1], [70, 3, 33]])
def test_the_same_bits_every_time_on_any_stream_and_in_graphs(n):
    c = Case(n, [700, 100, 1300], 16, 4, 128, 64, bits8=False).to_device()
    want = run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [run(c) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)
    outs, graphs = [torch.zeros_like(want) for _ in range(2)], []
    for out in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(c, out=out)
        graphs.append(g)
    for g in graphs:
        with torch.cuda.stream(torch.cuda.Stream()):
            g.replay()
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_keys_that_were_never_written_weigh_as_zeros():
    c = Case([1], [40], 8, 4, 64, 16, bits8=True)
    page = int(c.table[0, 1])
    c.scales[page], c.pages[page] = 0, torch.zeros_like(c.pages[page].float()).to(c.pages.dtype)
    c.rows[page] = 0
    want, tol = received(c)
    assert_close(run(c.to_device()), want, tol)


def test_extremes_of_an_8_bit_rows_scale():
    c = Case([1], [100], 8, 4, 128, 16, bits8=True, seed=4)
    for i, e in enumerate((-60, -30, 6)):
        c.scales[int(c.table[0, i])] = e + 127
        c.rows[int(c.table[0, i])] = c.pages[int(c.table[0, i])].double() * two_to(torch.tensor(e))
    want, tol = received(c)
    assert_close(run(c.to_device()), want, tol)


# ------------------------------------------------------------------------------------------------------------- many rows
MANY = {
    "one tile": ([16], [0], 8, 1, 128, 16),
    "a portion": ([150], [0], 10, 2, 128, 64),
    "behind others": ([77], [300], 8, 4, 64, 48),
    "ragged": ([40, 1, 0, 130, 33], [500, 129, 7, 0, 63], 8, 2, 128, 32),
    "one row too many": ([17], [400], 4, 4, 64, 7),
    "group of 5": ([52, 26], [260, 1000], 10, 2, 128, 64),
    "short requests": ([9] * 6, [3 * i for i in range(6)], 16, 4, 64, 16),
    "long": ([20], [5000], 4, 2, 128, 64),
}


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("step", MANY)
def test_many_rows(step, bits8):
    n, held, Hq, Hkv, dh, page = MANY[step]
    c = Case(n, held, Hq, Hkv, dh, page, seed=len(step), bits8=bits8).to_device()
    assert max(n) * Hq // Hkv > K().WEIGHTS_FEW
    want, tol = received(c)
    assert_close(run(c), want, tol)
    assert int(c.status) == 0


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("mask", MASKS)
def test_masks_and_scores_of_many_rows(mask, bits8):
    c = Case([150, 2, 40], [200, 300, 20], 8, 4, 64, 16, seed=5, bits8=bits8).to_device()
    a = _masks(c, mask)
    want, tol = received(c, **a)
    assert_close(run(c, **a), want, tol)


def test_only_the_last_rows_of_a_prompt():
    c = Case([100, 64], [50, 0], 8, 4, 64, 16, bits8=False).to_device()
    want, tol = received(c, rows=32)
    q, p = torch.cat([c.q[68:100], c.q[132:]]), torch.cat([c.positions[68:100], c.positions[132:]])
    c.q, c.positions, c.cu_q = q.contiguous(), p.contiguous(), torch.tensor([0, 32, 64], dtype=torch.int32).cuda()
    assert_close(run(c, max_count=32), want, tol)


def test_positions_in_any_order():
    c = Case([90], [0], 8, 2, 64, 16, bits8=False)
    c.positions = c.positions[torch.randperm(90, generator=torch.Generator().manual_seed(1))].contiguous()
    c.positions[7] = -3
    want, tol = received(c)
    assert_close(run(c.to_device()), want, tol)


def test_pages_that_a_window_has_left_behind_are_not_asked_for():
    c = Case([40, 1], [500, 300], 8, 4, 64, 16, bits8=False)
    for r in range(2):
        c.table[r, :(c.held[r] - 64) // 16] = -1
    want, tol = received(Case([40, 1], [500, 300], 8, 4, 64, 16, bits8=False), window=64)
    c.to_device()
    assert_close(run(c, window=64), want, tol)
    assert int(c.status) == 0


def test_a_few_rows_as_many_rows_gives_them(monkeypatch):
    """Either kernel on the same rows."""
    c = Case([2, 4], [300, 129], 8, 2, 128, 16, bits8=False).to_device()
    want, tol = received(c)
    few = run(c)
    monkeypatch.setattr(K(), "WEIGHTS_FEW", 0)
    many = run(c)
    assert_close(few, want, tol)
    assert_close(many, want, tol)


# ------------------------------------------------------------------------------------------- far places, calls side by side
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("n", [[1, 1], [40, 3]])
def test_pages_beyond_32_bits_of_bytes(n, bits8):
    """The same pages at the far end of a pool of 5 GB (10 GB) and at the near end of a small one."""
    c = Case(n, [200, 77], 16, 8, 128, 64, bits8=bits8).to_device()
    want, small = run(c), c.pages
    P, shift = 40000, 40000 - c.P
    far = torch.empty((P, *small.shape[1:]), dtype=small.dtype, device="cuda")
    assert far.numel() * far.element_size() > 2 ** 32
    far.view(torch.uint8)[shift:] = small.view(torch.uint8)
    c.pages = far
    if bits8:
        scales, c.scales = c.scales, torch.zeros((P, *c.scales.shape[1:]), dtype=torch.uint8, device="cuda")
        c.scales[shift:] = scales
    c.table = torch.where(c.table >= 0, c.table + shift, c.table)
    assert torch.equal(run(c), want)
    assert int(c.status) == 0


def test_two_calls_at_once():
    """Calls of both kinds on two streams, their scratch apart."""
    cases = [Case([1] * 6, [900, 3, 77, 2000, 512, 64], 16, 4, 128, 64, bits8=False, seed=1).to_device(), Case([90, 60], [700, 400], 16, 4, 128, 64, bits8=True, seed=2).to_device()]
    want = [run(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                outs[i].append(run(c))
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert all(torch.equal(g, w) for g in got)


def test_a_padded_batch():
    """Requests behind the last one have no tokens: their rows are what `add` says, and no table entry of theirs is looked at."""
    c = Case([1, 1, 1, 1], [100, 40, 9, 9], 8, 4, 64, 16, bits8=False)
    want, tol = received(c, width=120)
    want[2:], tol[2:] = 0, 0
    c.table[2:] = 1 << 30
    c.to_device()
    for count in (1, 30):  # either kernel
        c.status.zero_()
        got = run(c, width=120, cu_q=torch.tensor([0, 1, 2, 2, 2], dtype=torch.int32).cuda(), max_count=count)
        assert_close(got, want, tol)
        assert int(c.status) == 0


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("empty", [[0], [1], [0, 1, 2]])
@pytest.mark.parametrize("mask", [dict(window=64), dict(chunk=64), dict()])
def test_a_row_that_sees_nothing_beside_rows_that_do(mask, empty, few, bits8, monkeypatch):
    """Such a row's first key (0) is no key of the request's range, which a window or a chunk keeps short."""
    c = Case([3, 2], [1400, 700], 8, 2, 64, 16, bits8=bits8)
    for i in empty:
        c.positions[i] = -1 - 3 * i
    want, tol = received(c, **mask)
    c.to_device()
    if not few:
        monkeypatch.setattr(K(), "WEIGHTS_FEW", 0)
    assert_close(run(c, **mask), want, tol)
    assert int(c.status) == 0


@pytest.mark.parametrize("few", [True, False])
@pytest.mark.parametrize("empty", [[0], [2], [0, 1, 2]])
def test_a_row_that_sees_nothing_asks_for_no_page(empty, few, monkeypatch):
    """Pages that a window has left behind are no business of a row that sees no key at all."""
    c = Case([3, 2], [500, 300], 8, 4, 64, 16, bits8=False)
    for i in empty:
        c.positions[i] = -1
    want, tol = received(c, window=64)
    for r in range(2):
        c.table[r, :(c.held[r] - 64) // 16] = -1
    c.to_device()
    if not few:
        monkeypatch.setattr(K(), "WEIGHTS_FEW", 0)
    assert_close(run(c, window=64), want, tol)
    assert int(c.status) == 0


@pytest.mark.parametrize("bits8", [False, True])
def test_requests_in_several_launches_where_their_scratch_would_be_large(monkeypatch, bits8):
    """The same bits as from one launch, for every number of requests at a time."""
    c = Case([1, 2, 0, 1, 1], [900, 333, 0, 17, 640], 8, 2, 64, 64, bits8=bits8).to_device()
    plan = K().attention_weights_plan
    monkeypatch.setattr(K(), "attention_weights_plan", lambda *a: (*plan(*a)[:2], False))
    add = torch.rand((5, 2, 901), generator=torch.Generator().manual_seed(1)).cuda()
    want = run(c, width=901, add=add)
    assert_close(want, *received(c, width=901, add=add))
    splits, most, _ = plan(901, 10, 8, 148)
    one = 2 * splits * most * 8 * 4  # bytes of a request's scores
    for at_once, launches in ((1, 5), (2, 3), (3, 2), (5, 1), (0, 5)):
        monkeypatch.setattr(K(), "WEIGHTS_SCRATCH", at_once * one)
        before = K().launch_count()
        assert torch.equal(run(c, width=901, add=add), want)
        assert K().launch_count() == before + launches
    assert int(c.status) == 0


def test_scratch_is_bounded():
    """64 requests of a call that is sized for 131,072 keys: all of their scores would take 1.6 GB."""
    assert K().WEIGHTS_SCRATCH <= 512 << 20
    c = Case([1] * 64, [20 + i for i in range(64)], 40, 8, 128, 16, bits8=False).to_device()
    want, tol = received(c)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    got = run(c, max_kv=131072)
    assert torch.cuda.max_memory_allocated() - held <= K().WEIGHTS_SCRATCH + 2 * got.numel() * 4
    assert_close(got, want, tol)
    assert int(c.status) == 0


@pytest.mark.parametrize("sms", [1, 148])
@pytest.mark.parametrize("n", [[1, 1], [40, 3]])
def test_sums_with_room_for_more_keys_than_requests_have(n, sms, monkeypatch):
    """Every place is written once, behind the call's longest request, too: from `add`, from itself or with zeros."""
    c = Case(n, [300, 500], 8, 4, 64, 16, bits8=False).to_device()
    monkeypatch.setattr(K(), "sm_count", lambda: sms)
    for width in (501, 1024, 5000, 4096 * 3 + 1):
        want, tol = received(c, width=max(width, 540))
        want, tol = want[..., :width], tol[..., :width]
        add = torch.rand((2, 4, width), generator=torch.Generator().manual_seed(width)).cuda()
        if width > 540:
            assert_close(run(c, width=width), want, tol)
            assert_close(run(c, width=width, add=add), want + add.cpu().double(), tol + 2.0 ** -24 * (want + 1))
            there, before = add.clone(), K().launch_count()
            run(c, width=width, add=there, out=there)
            assert K().launch_count() == before + (1 if n[0] == 1 else 2)  # (and nothing to copy)
            assert_close(there, want + add.cpu().double(), tol + 2.0 ** -24 * (want + 1))
            assert torch.equal(there[..., 540:], add[..., 540:])
            assert int(c.status) == 0
        else:
            got = run(c, width=width, add=add, max_kv=600)  # (a request that has more gives nothing, and the status says so)
            c.status.zero_()
            assert_close(got[0], (want + add.cpu().double())[0], (tol + 2.0 ** -24 * (want + 1))[0])


# ------------------------------------------------------------------------------------ what only large steps reach, at small sizes
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("mask", [dict(), dict(window=64), dict(cap=5.0)])
def test_several_tiles_of_keys_a_block(monkeypatch, mask, bits8):
    """As on a device that holds two blocks: up to eight tiles of keys one after the other, some of which (window) no row sees."""
    c = Case([30, 40], [0, 900], 8, 4, 64, 16, seed=7, bits8=bits8)
    n = torch.arange(70)
    c.positions = torch.where(n % 2 == 0, c.positions, c.positions % 30).to(torch.int32)  # near the request's end and near its beginning
    want, tol = received(c, **mask)
    if mask.get("window"):
        assert float(want[1, :, 256:640].abs().max()) == 0
    c.to_device()
    monkeypatch.setattr(K(), "sm_count", lambda: 1)
    assert K()._weights_shares(2 * 4 * 8, 1, 2) == 1  # (and 2 * 4 * 8 tiles of keys on two places: eight a block)
    add = torch.rand(want.shape, generator=torch.Generator().manual_seed(1)).cuda()
    assert_close(run(c, **mask), want, tol)
    want, tol = received(c, add=add, **mask)
    assert_close(run(c, add=add, **mask), want, tol)
    assert int(c.status) == 0


@pytest.mark.parametrize("sms", [1, 148])
def test_more_than_32_tiles_of_rows_a_block(monkeypatch, sms):
    """16 heads on one: 38 tiles of rows, by one block or (several) shared by eight."""
    c = Case([300, 7], [0, 100], 16, 1, 64, 16, bits8=False, seed=3).to_device()
    monkeypatch.setattr(K(), "sm_count", lambda: sms)
    assert (K()._weights_shares(2 * 1 * 3, 38, 2 * sms) == 1) == (sms == 1)
    want, tol = received(c)
    assert_close(run(c), want, tol)
    assert int(c.status) == 0


@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("heads", [(8, 2), (16, 2), (32, 2)])
def test_ranges_of_more_keys_than_are_added_up_ahead(monkeypatch, bits8, heads):
    """One range of 2,500 keys a request: a thread adds up 20 of them."""
    monkeypatch.setattr(K(), "attention_weights_plan", lambda keys, *a: (1, -(-(keys + 16) // 16) * 16, False))
    c = Case([1, 1], [2500, 1100], *heads, 64, 64, bits8=bits8, seed=1).to_device()
    add = torch.rand((2, 2, 2501), generator=torch.Generator().manual_seed(1)).cuda()
    want, tol = received(c, add=add)
    assert_close(run(c, add=add), want, tol)
    assert_close(run(c), *received(c))
    assert int(c.status) == 0
