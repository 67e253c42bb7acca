"""The choice of the places that a cache keeps, moving the kept rows, and a decode loop that stays within its budget."""

import math

import pytest
import torch

from .budget_helpers import received
from .fp8_helpers import Case, assert_close, hold

pytestmark = pytest.mark.gpu
I32 = torch.int32


def K():
    from jax_llm_examples_b200.kernels import api

    return api


# ------------------------------------------------------------------------------------------------------------- choice
def choose(sums, lengths, keep, first=0, recent=0, most=None):
    R, H, _ = sums.shape
    most = max(keep) if most is None else most
    places, counts = torch.full((R, H, most), -7, dtype=I32, device="cuda"), torch.full((R,), -7, dtype=I32, device="cuda")
    status = torch.zeros(1, dtype=I32, device="cuda")
    K().kv_choose(sums.cuda(), torch.tensor(lengths, dtype=I32).cuda(), torch.tensor(keep, dtype=I32).cuda(), places, counts, status, first, recent)
    return places.cpu(), counts.tolist(), int(status)


def wanted(sums, L, n, first, recent):
    n = min(n, L)
    recent = min(recent, n)
    first = min(first, n - recent)
    forced = set(range(L - recent, L)) | set(range(first))
    value = [-math.inf if math.isnan(v) else v for v in sums[:L].tolist()]
    nan = [math.isnan(v) for v in sums[:L].tolist()]
    rest = sorted((j for j in range(L) if j not in forced), key=lambda j: (nan[j], -value[j], j))
    return sorted(forced | set(rest[:n - len(forced)]))


def check(sums, lengths, keep, first=0, recent=0):
    places, counts, status = choose(sums, lengths, keep, first, recent)
    assert status == 0
    for r, (L, n) in enumerate(zip(lengths, keep)):
        assert counts[r] == min(n, L)
        for h in range(sums.shape[1]):
            want = wanted(sums[r, h], L, n, first, recent)
            assert places[r, h].tolist() == want + [-1] * (places.shape[2] - len(want))


@pytest.mark.parametrize("width, lengths, keep", [
    (1, [1], [1]), (1, [0], [1]), (7, [7, 3], [4, 5]), (512, [512, 511, 0], [100, 511, 3]), (513, [513], [512]), (2049, [2049, 1000], [1, 999]), (5000, [4999, 17], [2500, 0]),
    (20001, [20001], [4096]), (40000, [40000], [39999]),
])
@pytest.mark.parametrize("first, recent", [(0, 0), (4, 0), (0, 64), (3, 1000)])
def test_choice(width, lengths, keep, first, recent):
    gen = torch.Generator().manual_seed(width)
    sums = torch.exp(2 * torch.randn((len(lengths), 2, width), generator=gen))
    sums[:, 1] = torch.round(4 * sums[:, 1]) / 4  # many ties
    check(sums, lengths, keep, first, recent)


def test_choice_over_all_numbers():
    gen = torch.Generator().manual_seed(5)
    sums = torch.randint(-2 ** 31, 2 ** 31, (2, 2, 3000), generator=gen, dtype=torch.int64).to(I32).view(torch.float32)  # any bits
    sums[0, 0, ::7] = math.nan
    sums[0, 1, ::5] = 0.0
    sums[0, 1, 1::5] = -0.0
    sums[1, 0] = 1.5
    sums[1, 1, ::3] = math.inf
    sums[1, 1, 1::3] = -math.inf
    check(sums, [3000, 2999], [1700, 1700], 2, 5)
    check(sums, [3000, 2999], [2990, 2500])


def test_choice_of_more_places_than_blocks_hold():
    gen = torch.Generator().manual_seed(6)
    sums = torch.randn((1, 1, 420000), generator=gen)
    sums[0, 0] = torch.round(sums[0, 0] * 100)
    check(sums, [419999], [60000], 4, 100)


def test_choice_refuses_on_the_device():
    sums = torch.arange(24.0).view(1, 2, 12)
    for lengths, keep, most, count in (([13], [5], 5, 5), ([-1], [5], 5, 0), ([12], [6], 5, 5), ([12], [-3], 5, 0)):
        places, counts, status = choose(sums, lengths, keep, most=most)
        assert status == 16 and counts == [count]
        assert places[0, 0].tolist() == list(range(12 - count, 12)) + [-1] * (most - count)


# ------------------------------------------------------------------------------------------------------------- moving
def pool(pages, H, page, dh, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    if dtype == torch.float8_e4m3fn:
        return torch.randint(0, 255, (pages, 2, H, page, dh), generator=gen, dtype=torch.uint8).cuda().view(dtype), \
            torch.randint(0, 255, (pages, 2, H, page), generator=gen, dtype=torch.uint8).cuda()
    return torch.randn((pages, 2, H, page, dh), generator=gen).to(dtype).cuda(), None


def tables(counts, page, order, width=None):
    per = [-(-c // page) for c in counts]
    t = torch.full((len(counts), width or max(max(per), 1)), -1, dtype=I32)
    for r, p in enumerate(per):
        t[r, :p] = torch.tensor([order.pop() for _ in range(p)], dtype=I32)
    return t


def bits(t):
    return t.view(torch.uint8).cpu()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("lengths, kept, H, page, dh", [
    ([1], [1], 1, 16, 64), ([100, 3, 40], [33, 3, 0], 3, 16, 64), ([1000, 517], [600, 517], 2, 64, 128), ([5000], [3000], 1, 48, 16), ([77], [50], 4, 7, 48),
    ([9000, 8000], [4100, 2100], 2, 32, 8),
])
def test_moving(in_place, dtype, lengths, kept, H, page, dh):
    if dh * torch.empty(0, dtype=dtype).element_size() % 16:
        pytest.skip("rows that are not whole 16 bytes are refused")
    gen = torch.Generator().manual_seed(1)
    total = sum(-(-t // page) for t in lengths + kept) + 2
    order = torch.randperm(total, generator=gen).tolist()
    src = tables(lengths, page, order)
    into = src if in_place else tables(kept, page, order)
    pages, scales = pool(total, H, page, dh, dtype)
    most, R = max(max(kept), 1) + 2, len(lengths)
    places = torch.full((R, H, most), -1, dtype=I32)
    for r in range(R):
        for h in range(H):
            places[r, h, :kept[r]] = torch.randperm(lengths[r], generator=gen)[:kept[r]].sort().values
    sums = torch.rand((R, H, max(lengths)), generator=gen)
    want, want_scales, want_sums = bits(pages), None if scales is None else scales.cpu(), torch.zeros_like(sums)
    old, old_scales = want.clone(), None if scales is None else scales.cpu()
    for r in range(R):
        for h in range(H):
            for i in range(kept[r]):
                j = int(places[r, h, i])
                s, d = (int(src[r, j // page]), j % page), (int(into[r, i // page]), i % page)
                want[d[0], :, h, d[1]] = old[s[0], :, h, s[1]]
                if scales is not None:
                    want_scales[d[0], :, h, d[1]] = old_scales[s[0], :, h, s[1]]
                want_sums[r, h, i] = sums[r, h, j]
    status = torch.zeros(1, dtype=I32, device="cuda")
    given = sums.cuda()
    out = None if in_place else torch.full((R, H, max(lengths)), math.nan, device="cuda")
    K().kv_compact(pages, src.cuda(), places.cuda(), torch.tensor(kept, dtype=I32).cuda(), status, into=None if in_place else into.cuda(), scales=scales, sums=given,
                   sums_out=out)
    assert torch.equal(bits(pages), want) and int(status) == 0  # every other row as it was
    assert scales is None or torch.equal(scales.cpu(), want_scales)
    assert torch.equal((given if in_place else out).cpu(), want_sums)


@pytest.mark.parametrize("in_place", [False, True])
def test_rows_without_a_page_are_left_out(in_place):
    pages, _ = pool(8, 2, 16, 64, torch.bfloat16)
    before = bits(pages)
    table = torch.tensor([[0, 1, 99]], dtype=I32).cuda()
    into = None if in_place else torch.tensor([[5, -1]], dtype=I32).cuda()
    places = torch.tensor([[[3, 20, 40], [5, 60, -2]]], dtype=I32).cuda()
    status = torch.zeros(1, dtype=I32, device="cuda")
    sums = torch.arange(96.0, device="cuda").view(1, 2, 48)
    out = torch.full((1, 2, 4), 7.0, device="cuda")
    K().kv_compact(pages, table, places, torch.tensor([3], dtype=I32).cuda(), status, into=into, sums=sums, sums_out=out)
    want, to = before.clone(), 0 if in_place else 5
    want[to, :, 0, 0], want[to, :, 0, 1], want[to, :, 1, 0] = before[0, :, 0, 3], before[1, :, 0, 4], before[0, :, 1, 5]
    assert torch.equal(bits(pages), want) and int(status) == 1
    assert out.tolist() == [[[3.0, 20.0, 40.0, 0.0], [53.0, 0.0, 0.0, 0.0]]]


def test_rows_do_not_move_back_in_place():
    pages, _ = pool(2, 1, 16, 64, torch.bfloat16)
    before = bits(pages)
    status = torch.zeros(1, dtype=I32, device="cuda")
    K().kv_compact(pages, torch.tensor([[1]], dtype=I32).cuda(), torch.tensor([[[4, 0, 9]]], dtype=I32).cuda(), torch.tensor([3], dtype=I32).cuda(), status)
    want = before.clone()
    want[1, :, 0, 0], want[1, :, 0, 2] = before[1, :, 0, 4], before[1, :, 0, 9]
    assert torch.equal(bits(pages), want) and int(status) == 1


def test_two_sessions_fork_from_one():
    """Pages may be read for several requests at once."""
    pages, _ = pool(6, 2, 16, 64, torch.bfloat16)
    before = bits(pages)
    status = torch.zeros(1, dtype=I32, device="cuda")
    places = torch.tensor([[[1, 9], [0, 30]], [[31, 31], [2, 3]]], dtype=I32)
    K().kv_compact(pages, torch.tensor([[0, 3], [0, 3]], dtype=I32).cuda(), places.cuda(), torch.tensor([2, 2], dtype=I32).cuda(), status,
                   into=torch.tensor([[1], [5]], dtype=I32).cuda())
    want = before.clone()
    for r, page in enumerate((1, 5)):
        for h in range(2):
            for i in range(2):
                j = int(places[r, h, i])
                want[page, :, h, i] = before[(0, 3)[j // 16], :, h, j % 16]
    assert torch.equal(bits(pages), want) and int(status) == 0


# ----------------------------------------------------------------------------------------------- together, as a decode loop
@pytest.mark.parametrize("bits8", [False, True])
@pytest.mark.parametrize("graph", [False, True])
def test_a_session_stays_within_its_budget(bits8, graph):
    """Weights of a prompt's last tokens, the cache cut to its budget, then tokens with weights and a cut each: step by step against the
    definitions, and attention over what was kept against attention over those rows alone."""
    budget, first, recent, page, Hq, Hkv, dh, steps = 40, 2, 8, 16, 8, 2, 64, 6
    c = Case([9, 9], [120, 61], Hq, Hkv, dh, page, seed=3, bits8=bits8)
    want, tol = received(c, width=160)
    c.to_device()
    sums = torch.zeros((2, Hkv, 160), device="cuda")
    run = lambda q, cu, pos, n: K().attention_weights(q, c.pages, c.table, cu, pos, sums, c.scale, 0, 0, 0.0, 1.0, c.status, 160, n, scales=c.scales, add=sums)  # noqa: E731
    run(c.q, c.cu_q, c.positions, 9)
    assert_close(sums, want, tol)
    keep = torch.full((2,), budget, dtype=I32, device="cuda")
    places, counts = torch.empty((2, Hkv, budget), dtype=I32, device="cuda"), torch.empty(2, dtype=I32, device="cuda")
    lengths = torch.tensor([129, 70], dtype=I32, device="cuda")
    gen = torch.Generator().manual_seed(9)
    tokens = (1.5 * torch.randn((steps, 2, Hq, dh), generator=gen)).to(torch.bfloat16).cuda()
    new = torch.randn((steps, 2, 2, Hkv, dh), generator=gen).to(torch.bfloat16).cuda()
    q, kv, cu, req = tokens[0].clone(), new[0].clone(), torch.tensor([0, 1, 2], dtype=I32).cuda(), torch.arange(2, dtype=I32).cuda()
    out = torch.empty_like(q)

    def cut():
        K().kv_choose(sums, lengths, keep, places, counts, c.status, first, recent)
        K().kv_compact(c.pages, c.table, places, counts, c.status, scales=c.scales, sums=sums)
        lengths.copy_(counts)

    def step():
        k, v = kv[0].contiguous(), kv[1].contiguous()
        if bits8:
            K().kv_store_fp8(k, v, c.pages, c.scales, c.table, req, lengths, c.status)
            K().attention_fp8(q, c.pages, c.scales, c.table, req, lengths, out, c.scale, 0, 0, 0.0, 1.0, c.status, 160)
        else:
            K().kv_store(k, v, c.pages, c.table, req, lengths, c.status)
            K().attention_generic(q, c.pages, c.table, req, lengths, out, c.scale, 0, 0, 0.0, 1.0, c.status)
        run(q, cu, lengths, 1)
        lengths.add_(1)
        cut()

    def rows_of():
        """Keys and values as numbers, [2, 2, Hkv, 160, dh]; their places beyond a request's are whatever lies there."""
        at = torch.arange(160, device="cuda")
        t = c.table[:, (at // page).clamp(max=c.table.shape[1] - 1)].long().clamp(min=0)
        raw = c.pages.view(torch.uint8)[t, :, :, at % page] if bits8 else c.pages[t, :, :, at % page]
        x = raw.view(torch.float8_e4m3fn).float() * torch.exp2(c.scales[t, :, :, at % page].float() - 127)[..., None] if bits8 else raw.float()
        return x.double().permute(0, 2, 3, 1, 4)

    cut()
    assert lengths.tolist() == [budget, budget]
    g = None
    for i in range(steps):
        q.copy_(tokens[i])
        kv.copy_(new[i].transpose(0, 1))
        sums_before, rows_before = sums.clone(), rows_of()
        L = int(lengths[0])
        if graph and g is None:
            saved = [t.clone() for t in (c.pages.view(torch.uint8), sums, lengths)] + ([c.scales.clone()] if bits8 else [])
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            for t, s in zip([c.pages.view(torch.uint8), sums, lengths] + ([c.scales] if bits8 else []), saved):
                t.copy_(s)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                step()
        if g is not None:
            g.replay()
        else:
            step()
        # the definitions, on what the step began with
        rows = rows_before.clone()
        rows[:, :, :, L] = hold(new[i].cpu())[0].cuda() if bits8 else new[i].double()
        k, v = rows[:, 0, :, :L + 1], rows[:, 1, :, :L + 1]
        s = torch.einsum("rhgd,rhld->rhgl", tokens[i].double().view(2, Hkv, Hq // Hkv, dh), k) * c.scale
        w = torch.softmax(s, -1)
        o = torch.einsum("rhgl,rhld->rhgd", w, v).reshape(2, Hq, dh)
        # weights rounded to 16 bits for the product (2^-8), the output to bfloat16 (2^-8)
        assert float((out.double() - o).abs().max()) <= 2.0 ** -7 * float(v.abs().max())
        total = sums_before.double()
        total[:, :, :L + 1] += w.sum(2)
        for r in range(2):
            for h in range(Hkv):
                kept = places[r, h].long()
                assert kept.tolist() == sorted(kept.tolist()) and kept[:first].tolist() == list(range(first)) and kept[-recent:].tolist() == list(range(L + 1 - recent, L + 1))
                dropped = [j for j in range(L + 1) if j not in set(kept.tolist())]
                chosen = kept[first:-recent]
                # sums as near as the kernel's error may be taken either way
                assert float(total[r, h, dropped].max()) <= float(total[r, h, chosen].min()) * (1 + 2.0 ** -14)
                assert torch.allclose(sums[r, h, :budget].double(), total[r, h, kept], rtol=2.0 ** -14, atol=0)
                assert float(sums[r, h, budget:].abs().max()) == 0
                assert torch.equal(rows_of()[r, :, h, :budget], rows[r, :, h, kept])
    assert lengths.tolist() == [budget, budget] and int(c.status) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_the_same_bits_on_another_stream(dtype):
    gen = torch.Generator().manual_seed(2)
    sums = torch.rand((2, 3, 4000), generator=gen).cuda()
    lengths, keep = torch.tensor([4000, 3777], dtype=I32).cuda(), torch.tensor([1000, 2000], dtype=I32).cuda()
    got = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            pages, scales = pool(300, 3, 64, 64, dtype)
            places, counts, status = torch.empty((2, 3, 2000), dtype=I32, device="cuda"), torch.empty(2, dtype=I32, device="cuda"), torch.zeros(1, dtype=I32, device="cuda")
            table = torch.arange(200, dtype=I32, device="cuda").view(2, 100)
            K().kv_choose(sums, lengths, keep, places, counts, status, 4, 100)
            moved = sums.clone()
            K().kv_compact(pages, table, places, counts, status, scales=scales, sums=moved)
            got.append((bits(pages), places.cpu(), moved.cpu(), int(status)))
    assert all(torch.equal(a, b) if isinstance(a, torch.Tensor) else a == b == 0 for a, b in zip(*got))


@pytest.mark.parametrize("in_place", [False, True])
def test_moving_beyond_32_bits_of_bytes(in_place):
    P, H, page, dh = 33000, 8, 64, 128
    pages = torch.empty((P, 2, H, page, dh), dtype=torch.bfloat16, device="cuda")
    assert pages.numel() * 2 > 2 ** 32
    used = [P - 1, 2, P - 7]
    for p in used + [P - 3, 5]:
        pages[p] = torch.randn((2, H, page, dh), device="cuda").to(torch.bfloat16)
    table = torch.tensor([used], dtype=I32).cuda()
    into = None if in_place else torch.tensor([[P - 3, 5]], dtype=I32).cuda()
    gen = torch.Generator().manual_seed(1)
    places = torch.stack([torch.randperm(3 * page, generator=gen)[:100].sort().values for _ in range(H)])[None].to(I32)
    rows = pages[used].permute(1, 2, 0, 3, 4).reshape(2, H, 3 * page, dh)
    want = torch.stack([rows[:, h, places[0, h].long().cuda()] for h in range(H)], 1)
    status = torch.zeros(1, dtype=I32, device="cuda")
    K().kv_compact(pages, table, places.cuda(), torch.tensor([100], dtype=I32).cuda(), status, into=into)
    to = used[:2] if in_place else [P - 3, 5]
    got = pages[to].permute(1, 2, 0, 3, 4).reshape(2, H, 2 * page, dh)[:, :, :100]
    assert torch.equal(got, want) and int(status) == 0


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("counts, most, out_width, moved, summed", [
    ([5, 2], 3, 8, [3, 2], [3, 2]),  # more rows than `places` has
    ([-1, 1], 3, 8, [0, 1], [0, 1]),
    ([3, 1], 3, 2, [3, 1], [2, 1]),  # more sums than `sums_out` has
    ([1, 0], 0, 8, [0, 0], [0, 0]),  # no places at all
])
def test_counts_that_their_arrays_do_not_hold_raise_the_status(in_place, counts, most, out_width, moved, summed):
    pages, _ = pool(6, 2, 16, 64, torch.bfloat16)
    before = bits(pages)
    table = torch.tensor([[0], [1]], dtype=I32)
    into = table if in_place else torch.tensor([[4], [5]], dtype=I32)
    places = torch.tensor([[2, 5, 7], [3, 4, 15]], dtype=I32).expand(2, 2, 3)[:, :, :most].contiguous()  # of each head
    sums = torch.rand((2, 2, 16), generator=torch.Generator().manual_seed(1)).cuda()
    out = torch.full((2, 2, out_width), math.nan, device="cuda")
    status = torch.zeros(1, dtype=I32, device="cuda")
    K().kv_compact(pages, table.cuda(), places.cuda(), torch.tensor(counts, dtype=I32).cuda(), status, into=None if in_place else into.cuda(), sums=sums, sums_out=out)
    assert int(status) == 16
    want, want_sums = before.clone(), torch.zeros((2, 2, out_width))
    for r in range(2):
        for h in range(2):
            for i in range(moved[r]):
                want[into[r, 0], :, h, i] = before[table[r, 0], :, h, places[r, h, i]]
            for i in range(summed[r]):
                want_sums[r, h, i] = sums[r, h, places[r, h, i]].cpu()
    assert torch.equal(bits(pages), want) and torch.equal(out.cpu(), want_sums)


@pytest.mark.parametrize("requests, H, width", [(37, 4, 8192), (1, 1, 100001)])
def test_choice_of_as_many_places_as_threads_hold(requests, H, width):
    """13 to 16 sums a thread: a block a row, and sixteen."""
    gen = torch.Generator().manual_seed(width)
    sums = torch.exp(1.5 * torch.randn((requests, H, width), generator=gen) - 5)
    sums[:, ::2] = sums[:, ::2].to(torch.bfloat16).float()
    sums[0, 0, ::3] = 0.0
    check(sums, [width - 211 * i for i in range(requests)], [width // 4 + 31 * i for i in range(requests)], 4, 256)
