"""Low-rank adapters, host side: the plan of a step's rows, and refusals before anything is launched."""

import pytest
import torch

from jax_llm_examples_b200.kernels import api as K


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


@pytest.mark.parametrize("of_row", [[0], [-1], [], [2, 0, 2, -1, 0], [1] * 16, [1] * 17, [3] * 200 + [0] * 64 + [-1] * 65 + [2], [5, 4, 3, 2, 1, 0] * 11])
def test_a_plan_holds_every_row_once(of_row):
    plan = K.adapter_plan(of_row, 6, device="cpu")
    order, tiles = plan.order.tolist(), plan.tiles.tolist()
    assert sorted(order) == list(range(len(of_row))) and plan.rows == len(of_row)
    seen = []
    for e, first, count in tiles:
        assert 0 < count <= plan.tile_rows
        rows = order[first:first + count]
        assert all(of_row[n] == e for n in rows) and rows == sorted(rows)
        seen += rows
    assert sorted(seen) == list(range(len(of_row)))
    # as few tiles as the rows' adapters allow
    assert len(tiles) == sum(-(-of_row.count(e) // plan.tile_rows) for e in set(of_row))


@pytest.mark.parametrize("of_row, adapters", [([0, 6], 6), ([-2], 6), ([0], 0)])
def test_a_plan_refuses_unknown_adapters(of_row, adapters):
    with pytest.raises(K.KernelError, match="adapter_plan"):
        K.adapter_plan(of_row, adapters, device="cpu")


def _args(**change):
    a = dict(x=torch.zeros(5, 32), a=torch.zeros(3, 4, 32), b=torch.zeros(3, 16, 4), plan=K.adapter_plan([0, 1, -1, 1, 2], 3, device="cpu"), y=torch.zeros(5, 16))
    return {**a, **change}


@pytest.mark.parametrize("change, match", [
    (dict(), "not on the GPU"),
    (dict(x=torch.zeros(5, 32, dtype=torch.bfloat16)), "type"),
    (dict(out=torch.zeros(5, 16, dtype=torch.bfloat16)), "type"),
    (dict(x=torch.zeros(5, 33)), "x must be"),
    (dict(x=torch.zeros(32, 5).T), "x must be"),
    (dict(y=torch.zeros(4, 16)), "y must be"),
    (dict(y=torch.zeros(5, 17)), "y must be"),
    (dict(out=torch.zeros(1, 16).expand(5, 16)), "out must be"),
    (dict(a=torch.zeros(2, 4, 32)), "matrices"),
    (dict(b=torch.zeros(3, 16, 5)), "matrices"),
    (dict(a=torch.zeros(4, 32)), "matrices"),
    (dict(a=torch.zeros(3, 257, 32), b=torch.zeros(3, 16, 257)), "rank"),
    (dict(a=torch.zeros(3, 0, 32), b=torch.zeros(3, 16, 0)), "rank"),
    (dict(plan=K.adapter_plan([0] * 4, 3, device="cpu")), "plan"),
    (dict(plan=K.adapter_plan([0] * 5, 2, device="cpu")), "plan"),
    (dict(scale=torch.ones(2)), "scale"),
    (dict(scale=torch.ones(3, dtype=torch.float64)), "scale"),
    (dict(ranks=torch.ones(3)), "ranks"),
    (dict(y=torch.zeros(5, 16, dtype=torch.float16)), "type"),
])
def test_refusals(no_launch, change, match):
    with pytest.raises(K.KernelError, match=match):
        K.adapter_add(**_args(**change))


def test_out_may_be_y_but_no_part_of_an_operand(no_launch, monkeypatch):
    monkeypatch.setattr(K, "_placed", lambda *a: -1)  # as if the tensors were on the device
    wide = torch.zeros(5, 64)
    for change in (dict(out=wide[:, 8:24], y=wide[:, :16]), dict(out=wide[:, 40:56], x=wide[:, 16:48]), dict(x=wide[:, :32], y=wide[:, 24:40]),
                   dict(y=torch.as_strided(wide, (5, 16), (64, 1)), out=torch.as_strided(wide, (5, 16), (16, 1)))):
        with pytest.raises(K.KernelError, match="shares memory"):
            K.adapter_add(**_args(**change))
    assert not K._overlap(wide[:, :16], wide[:, 16:48]) and K._overlap(wide[:, :17], wide[:, 16:48])
    assert not K._overlap(wide[:2], wide[2:]) and K._overlap(wide[:3], wide[2:])
    assert not K._overlap(wide[:, 48:], wide[:, :48]) and K._overlap(wide[1:, 40:], wide[:, 41:])


def test_rows_without_an_adapter_do_not_make_the_tiles_larger():
    """A tile's size goes by the adapters' rows: decoding sessions keep tiles of 16 though many of them have none."""
    assert K.adapter_plan([-1] * 17 + list(range(24)), 24, device="cpu").tile_rows == 16
    assert K.adapter_plan([-1] * K.ADAPTER_BARE + [0], 24, device="cpu").tile_rows == 16
    assert K.adapter_plan([-1] * (K.ADAPTER_BARE + 1) + [0], 24, device="cpu").tile_rows == 64  # (a portion's)
    assert K.adapter_plan([-1] * 17 + [3] * 17, 24, device="cpu").tile_rows == 64
    plan = K.adapter_plan([-1] * 40 + [0, 1, 1], 2, device="cpu")
    assert plan.tiles.tolist() == [[-1, 0, 16], [-1, 16, 16], [-1, 32, 8], [0, 40, 1], [1, 41, 2]]
