"""Low-rank adapters of many requests beside a shared projection, against the definition in 64 bits.

What a result may be off by: the sums of K products and of r, in 32 bits, by 2^-23 of the magnitudes' sum an addition (the tensor
cores cut, not round); between the products bfloat16 operands pass as two bfloat16 numbers, off by 2^-16, for 32-bit outputs as
three, off by 2^-24; the last rounding by 2^-8 or 2^-24 of the result."""

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def K():
    from jax_llm_examples_b200.kernels import api

    return api


class Step:
    def __init__(self, of_row, E, r, k, n, dtype=BF, out_dtype=BF, mixed=False, seed=0, wide=0):
        gen = torch.Generator().manual_seed(seed)
        N = len(of_row)
        rand = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
        rows = lambda w, t: torch.cat([rand(N, w) * torch.exp(rand(N, 1)), rand(N, wide)], 1).to(t).cuda()[:, :w]  # noqa: E731
        self.of_row, self.x, self.y = of_row, rows(k, dtype), rows(n, out_dtype)
        self.a, self.b = (rand(E, r, k) * k ** -0.5).to(dtype).cuda(), (rand(E, n, r)).to(dtype).cuda()
        self.scale = (0.5 + torch.rand(E, generator=gen)).cuda()
        self.ranks = torch.tensor([max(0, r - 5 * (e % 4)) for e in range(E)], dtype=torch.int32).cuda() if mixed else None
        self.plan = K().adapter_plan(of_row, E)

    def run(self, out=None):
        out = torch.full_like(self.y, float("nan")) if out is None else out
        K().adapter_add(self.x, self.a, self.b, self.plan, self.y, out, scale=self.scale, ranks=self.ranks)
        return out

    def want(self):
        """(The definition, how far a result may be off.)"""
        y = self.y.double()
        out, off = y.clone(), torch.zeros_like(y)
        k, r = self.a.shape[2], self.a.shape[1]
        between = 0.0 if self.x.dtype == F32 else 2.0 ** -24 if self.y.dtype == F32 else 2.0 ** -16
        for n, e in enumerate(self.of_row):
            if e < 0:
                continue
            m = r if self.ranks is None else int(self.ranks[e])
            a, b, x, s = self.a[e, :m].double(), self.b[e, :, :m].double(), self.x[n].double(), self.scale[e].double()
            out[n] += s * (b @ (a @ x))
            off[n] = (b.abs() @ (a.abs() @ x.abs())) * s * ((k + r + 4) * 2.0 ** -23 + between)
        rounds = 2.0 ** -8 if self.y.dtype == BF else 2.0 ** -23  # (32 bits: the addition of y, too)
        return out, off * (1 + rounds) + rounds * out.abs() + (2.0 ** -24 * y.abs())

    def check(self, got):
        want, off = self.want()
        assert bool(((got.double() - want).abs() <= off).all()), float(((got.double() - want).abs() / off).max())
        none = torch.tensor([e < 0 for e in self.of_row]).cuda()
        assert torch.equal(got[none], self.y[none])


ROWS = {
    "one": [0], "bare": [-1], "few": [2, 0, 2, -1, 0], "tile": [1] * 16, "tile and one": [1] * 17, "own each": list(range(24)), "shared": [0, 1, 2, -1] * 16,
    "portions": [3] * 100 + [0] * 64 + [-1] * 33 + [2] * 31 + [1], "steps beside a portion": [4] * 129 + [0, 1, 2, 3, -1, 1, 2],
}


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("r, k, n, dtype, out_dtype", [
    (16, 256, 320, BF, BF), (8, 72, 40, BF, F32), (64, 1000, 264, BF, F32), (24, 520, 1032, BF, BF), (128, 264, 128, BF, BF), (200, 136, 96, BF, F32),
    (256, 512, 64, BF, BF), (13, 100, 77, BF, BF), (1, 8, 8, BF, F32), (4, 129, 33, F32, F32), (64, 512, 300, F32, F32), (16, 64, 64, F32, BF), (8, 1, 1, BF, BF),
    (32, 2048, 24, BF, BF),
])
def test_rows_of_many_adapters(rows, r, k, n, dtype, out_dtype):
    step = Step(ROWS[rows], 24, r, k, n, dtype, out_dtype, seed=r + k)
    step.check(step.run())


@pytest.mark.parametrize("r", [8, 16, 40, 128, 13])
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_ranks_of_their_own_and_nothing_read_behind_them(r, out_dtype):
    step = Step(ROWS["steps beside a portion"], 5, r, 264, 136, BF, out_dtype, mixed=True, seed=r)
    for e in range(5):
        step.a[e, int(step.ranks[e]):] = float("nan")
        step.b[e, :, int(step.ranks[e]):] = float("inf")
    step.check(step.run())


@pytest.mark.parametrize("wide", [8, 3])
@pytest.mark.parametrize("rows", ["few", "portions"])
def test_column_ranges_of_wider_rows_and_in_place(wide, rows):
    step = Step(ROWS[rows], 6, 16, 256, 160, wide=wide)
    want, off = step.want()
    base = step.y._base if step.y._base is not None else step.y
    behind = base[:, 160:].clone()
    K().adapter_add(step.x, step.a, step.b, step.plan, step.y, scale=step.scale)
    assert bool(((step.y.double() - want).abs() <= off).all())
    assert torch.equal(base[:, 160:], behind)


def test_the_first_of_split_partials():
    step = Step(ROWS["shared"], 4, 16, 512, 256, BF, F32)
    parts = torch.stack([step.y, torch.randn_like(step.y)])
    other, step.y = parts[1].clone(), parts[0]
    want, off = step.want()
    K().adapter_add(step.x, step.a, step.b, step.plan, parts[0], scale=step.scale)
    assert bool(((parts[0].double() - want).abs() <= off).all()) and torch.equal(parts[1], other)


@pytest.mark.parametrize("dtype, r", [(BF, 16), (BF, 13), (F32, 8)])
def test_what_is_not_finite_stays_in_its_row(dtype, r):
    step = Step([0, 1, 0, 2, 1, -1], 3, r, 264, 136, dtype, dtype)
    step.x[0, 5], step.x[1, 3] = float("nan"), float("inf")
    step.b[2] = float("nan")
    got = step.run()
    assert bool(got[0].isnan().all()) and bool(got[3].isnan().all()) and not bool(got[1].isfinite().any())
    for n in (2, 4, 5):
        assert bool(got[n].isfinite().all())


@pytest.mark.parametrize("r, dtype", [(16, BF), (64, BF), (5, F32)])
def test_the_same_bits_every_time_on_any_stream_and_in_a_graph(r, dtype):
    step = Step(ROWS["portions"], 4, r, 520, 264, dtype, dtype)
    want = step.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step.run() for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)
    outs = [torch.zeros_like(want) for _ in range(2)]
    graphs = []
    for out in outs:  # two graphs, replayed beside each other
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step.run(out)
        graphs.append(g)
    for g in graphs:
        with torch.cuda.stream(torch.cuda.Stream()):
            g.replay()
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_no_rows_and_counted_launches():
    step = Step([], 2, 8, 64, 64)
    before = K().launch_count()
    assert step.run().shape == (0, 64) and K().launch_count() == before
    Step([0, 1], 2, 8, 64, 64).run()
    assert K().launch_count() == before + 1
    Step([0, 1], 2, 8, 63, 64).run()
    assert K().launch_count() == before + 3


@pytest.mark.parametrize("rows, dtype, out_dtype, partials", [("few", BF, BF, True), ("shared", BF, F32, False), ("steps beside a portion", BF, F32, True),
                                                             ("portions", BF, BF, False), ("few", F32, F32, True)])
def test_beside_a_projection(rows, dtype, out_dtype, partials):
    """The part that does both: the projection's own kernels for few and for many rows, adapters on its result or its partials."""
    from jax_llm_examples_b200.parts import Adapters, Runtime, StepContext, Workspace, adapted_linear, linear
    from jax_llm_examples_b200.parts.base import Rows

    of_row = ROWS[rows] * (3 if rows == "portions" else 1)  # (over 256 rows: the library's product)
    step = Step(of_row, 6, 16, 1024, 512, dtype, out_dtype, seed=3)
    w = (torch.randn(512, 1024, generator=torch.Generator().manual_seed(4)) * 1024 ** -0.5).to(dtype).cuda()
    N, t = len(of_row), torch.zeros(len(of_row), dtype=torch.int32, device="cuda")
    ctx = StepContext(runtime=Runtime(dtype, torch.device("cuda")), n_tokens=N, n_requests=1, token_ids=t, positions=t, req_of_token=t, cu_q=t[:2], q_start=t[:1],
                      kv_len=t[:1], slot_ids=t[:1], logit_rows=t[:0], n_logit_rows=0, status=t[:1].clone(), workspace=Workspace(torch.device("cuda")))
    plain = lambda r: (r.data.float().sum(0) if r.data.dim() == 3 else r.data) if isinstance(r, Rows) else r  # noqa: E731
    step.y = plain(linear(ctx, step.x, w, out_dtype, partials))  # what the adapters are added to
    want, off = step.want()
    got = plain(adapted_linear(ctx, step.x, w, Adapters(step.a, step.b, step.scale), step.plan, out_dtype, partials))
    # (partials: up to eight slices are added here, each addition off by half a step of the largest)
    assert bool(((got.double() - want).abs() <= off + 8 * 2.0 ** -24 * (want.abs() + step.y.double().abs() + 8)).all())


def test_matrices_beyond_32_bits():
    """The last of many adapters, whose matrices lie 2^31 entries behind the first one's.  All entries are -1, 0 or 1: every sum is a whole
    number below 2^24, which 32 bits, and three bfloat16 numbers, hold."""
    E, r, k, n = 66, 64, 520000, 512
    a, b = torch.empty((E, r, k), dtype=BF, device="cuda"), torch.zeros((E, n, r), dtype=BF, device="cuda")
    assert a.numel() > 2 ** 31
    gen = torch.Generator().manual_seed(1)
    ones = lambda *s: torch.randint(-1, 2, s, generator=gen)  # noqa: E731
    a[-1], b[-1] = ones(r, k).to(BF).cuda(), ones(n, r).to(BF).cuda()
    for of_row in ([65], [65] * 40):
        x, y = ones(len(of_row), k).to(BF).cuda(), ones(len(of_row), n).float().cuda()
        out = torch.empty_like(y)
        K().adapter_add(x, a, b, K().adapter_plan(of_row, E), y, out)
        low = torch.cat([a[-1, i:i + 8].double() @ x.double().T for i in range(0, r, 8)]).T
        want = y.double() + low @ b[-1].double().T
        assert float(want.abs().max()) < 2 ** 24 and torch.equal(out.double(), want)


def test_two_calls_at_once():
    steps = [Step(ROWS["portions"], 4, 16, 520, 264, BF, BF, seed=1), Step(ROWS["few"], 3, 13, 99, 77, BF, F32, seed=2)]  # (one with scratch)
    want = [s.run() for s in steps]
    streams, outs = [torch.cuda.Stream() for _ in steps], [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for i, (step, s) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(s):
                outs[i].append(step.run())
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert all(torch.equal(g, w) for g in got)


@pytest.mark.parametrize("rows", ["few", "tile and one", "portions"])
@pytest.mark.parametrize("r, k, n, dtype, out_dtype", [(16, 256, 320, BF, BF), (64, 1000, 264, BF, F32), (13, 264, 136, BF, BF), (200, 136, 96, BF, F32), (8, 100, 77, BF, BF),
                                                       (40, 264, 136, BF, BF), (16, 64, 64, F32, F32)])
def test_infinite_entries_of_b_give_infinities(rows, r, k, n, dtype, out_dtype):
    """An entry of a column: the result is infinite, whatever the rows between the products pass as; two of opposite effect: NaN."""
    step = Step(ROWS[rows], 6, r, k, n, dtype, out_dtype, seed=r)
    step.x.abs_()
    step.a.abs_()  # (so no number between the products is near 0)
    for col, rank, value in ((0, 0, "inf"), (3, r - 1, "-inf"), (n - 1, r // 2, "inf"), (17, 1, "inf"), (17, 2, "-inf"), (20, 4, "nan")):
        step.b[:, col, rank] = float(value)
    want, off = step.want()
    got, sure = step.run(), want.isfinite()
    assert bool(want[:, 0].isinf().any()) and bool(want[:, 17].isnan().any())
    assert torch.allclose(got[~sure].double(), want[~sure], rtol=0, atol=0, equal_nan=True)
    assert bool(((got.double() - want).abs() <= off)[sure].all())


@pytest.mark.parametrize("rows", ["few", "tile and one", "portions"])
@pytest.mark.parametrize("r, k, n, dtype, out_dtype, mixed", [(16, 256, 320, BF, BF, True), (64, 1000, 264, BF, F32, True), (13, 264, 136, BF, BF, False), (200, 136, 96, BF, F32, False),
                                                              (8, 100, 77, BF, BF, True), (24, 264, 136, BF, BF, True), (24, 264, 136, BF, BF, False), (7, 64, 64, F32, F32, True)])
def test_infinite_rows_meet_no_rank_that_is_not_there(rows, r, k, n, dtype, out_dtype, mixed):
    """Ranks behind an adapter's own are not zeros that an infinity is multiplied with: infinite results stay infinite, and an adapter of
    rank 0 changes nothing."""
    step = Step(ROWS[rows], 6, r, k, n, dtype, out_dtype, mixed=mixed, seed=r)
    if mixed:
        step.ranks[::3] = 0
        step.ranks[1::3] = 1
        step.ranks[2::3] = r - 3
    step.a.abs_()
    step.b.abs_()
    step.x[::2, 3] = float("inf")
    want, off = step.want()
    got, sure = step.run(), want.isfinite()
    assert bool(want.isposinf().any()) and not bool(want.isnan().any())
    assert torch.equal(got[~sure].double(), want[~sure])
    assert bool(((got.double() - want).abs() <= off)[sure].all())
    if mixed:
        none = (step.ranks[torch.tensor(step.of_row).clamp(min=0)] == 0).cuda()
        assert torch.equal(got[none], step.y[none])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("out_dtype", [BF, F32])
def test_many_rows_without_an_adapter_beside_single_ones(out_dtype, in_place):
    step = Step([-1] * 77 + list(range(24)) + [-1] * 3, 24, 32, 264, 136, BF, out_dtype)
    assert step.plan.tile_rows == 16
    want, off = step.want()
    got = step.y.clone() if in_place else torch.full_like(step.y, float("nan"))
    K().adapter_add(step.x, step.a, step.b, step.plan, got if in_place else step.y, got, scale=step.scale)
    step.check(got)
