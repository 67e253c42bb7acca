"""A cache kept to a budget, host side: refusals before anything is launched, and the rules on sizes."""

import pytest
import torch

from jax_llm_examples_b200.kernels import api as K

from .fp8_helpers import Case


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


I32 = torch.int32


def _weights(**change):
    c = Case([3], [5], 4, 2, 64, 16, device="cpu", bits8=False)
    a = dict(q=c.q, pages=c.pages, block_table=c.table, cu_q=c.cu_q, positions=c.positions, out=torch.zeros(1, 2, 8), scale=0.125, chunk=0, window=0,
             attn_scale=0.0, floor_scale=1.0, status=c.status, max_kv_len=8, max_count=3)
    return {**a, **change}


@pytest.mark.parametrize("change, match", [
    (dict(), "not on the GPU"),
    (dict(q=torch.zeros(3, 4, 64)), "bfloat16"),
    (dict(q=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), "disagree"),
    (dict(pages=torch.zeros(4, 2, 2, 16, 64)), "pages"),
    (dict(scales=torch.zeros((4, 2, 2, 16), dtype=torch.uint8)), "float8"),
    (dict(block_table=torch.zeros((1, 2), dtype=torch.int64)), "block table"),
    (dict(cu_q=torch.zeros(1, dtype=I32)), "cu_q"),
    (dict(positions=torch.zeros(3)), "positions"),
    (dict(out=torch.zeros(1, 2, 8, dtype=torch.bfloat16)), "out"),
    (dict(out=torch.zeros(2, 2, 8)), "out"),
    (dict(add=torch.zeros(1, 2, 9)), "add"),
    (dict(add=torch.zeros(1, 2, 8, dtype=torch.float64)), "add"),
    (dict(max_kv_len=0), "keys"),
    (dict(max_count=0), "tokens"),
    (dict(sink=torch.zeros(3)), "sink"),
    (dict(slopes=torch.zeros(4, dtype=torch.bfloat16)), "slopes"),
    (dict(q=torch.zeros((3, 64, 4), dtype=torch.bfloat16).transpose(1, 2)), "contiguous"),
])
def test_weights_refuse(no_launch, change, match):
    with pytest.raises(K.KernelError, match=match):
        K.attention_weights(**_weights(**change))


def test_weights_are_not_added_over_shifted_memory(no_launch):
    both = torch.zeros(24)
    with pytest.raises(K.KernelError, match="add"):
        K.attention_weights(**_weights(out=both[:16].view(1, 2, 8), add=both[4:20].view(1, 2, 8)))


@pytest.mark.parametrize("keys", [1, 15, 16, 700, 8192, 30000, 131072])
@pytest.mark.parametrize("pairs", [1, 8, 64, 512])
@pytest.mark.parametrize("rows", [1, 8, 16])
def test_ranges_hold_all_keys(keys, pairs, rows):
    splits, most, fits = K.attention_weights_plan(keys, pairs, rows, 148)
    assert 1 <= splits <= 16 and most % K.WEIGHTS_KEYS == 0
    # a first key anywhere within a tile
    assert splits * most >= keys + K.WEIGHTS_KEYS - 1 and fits == (most * 8 * -(-rows // 2) <= K.WEIGHTS_HELD)


def _choose(**change):
    a = dict(sums=torch.zeros(2, 3, 10), lengths=torch.ones(2, dtype=I32), keep=torch.ones(2, dtype=I32), places=torch.zeros((2, 3, 4), dtype=I32),
             counts=torch.zeros(2, dtype=I32), status=torch.zeros(1, dtype=I32))
    return {**a, **change}


@pytest.mark.parametrize("change, match", [
    (dict(), "not on the GPU"),
    (dict(sums=torch.zeros(2, 3, 10, dtype=torch.bfloat16)), "sums"),
    (dict(sums=torch.zeros(2, 30)), "sums"),
    (dict(lengths=torch.ones(1, dtype=I32)), "lengths"),
    (dict(keep=torch.ones(2)), "keep"),
    (dict(places=torch.zeros((2, 2, 4), dtype=I32)), "places"),
    (dict(places=torch.zeros((2, 3, 4))), "places"),
    (dict(counts=torch.zeros(1, dtype=I32)), "counts"),
    (dict(first=-1), "first"),
    (dict(recent=-1), "last"),
    (dict(sums=torch.zeros(2, 10, 3).transpose(1, 2)), "contiguous"),
])
def test_choosing_refuses(no_launch, change, match):
    with pytest.raises(K.KernelError, match=match):
        K.kv_choose(**_choose(**change))


def _compact(**change):
    a = dict(pages=torch.zeros(4, 2, 3, 16, 64), block_table=torch.zeros((2, 2), dtype=I32), places=torch.zeros((2, 3, 4), dtype=I32),
             counts=torch.zeros(2, dtype=I32), status=torch.zeros(1, dtype=I32))
    return {**a, **change}


@pytest.mark.parametrize("change, match", [
    (dict(), "not on the GPU"),
    (dict(pages=torch.zeros(4, 3, 16, 64)), "pages"),
    (dict(pages=torch.zeros(4, 2, 3, 16, 64).to(torch.float8_e4m3fn)), "scales"),
    (dict(scales=torch.zeros((4, 2, 3, 16), dtype=torch.uint8)), "scales"),
    (dict(pages=torch.zeros(4, 2, 3, 16, 6, dtype=torch.bfloat16)), "16 bytes"),
    (dict(places=torch.zeros((2, 2, 4), dtype=I32)), "places"),
    (dict(places=torch.zeros((2, 3, 4), dtype=torch.int64)), "places"),
    (dict(counts=torch.zeros(1, dtype=I32)), "counts"),
    (dict(block_table=torch.zeros((1, 2), dtype=I32)), "block tables"),
    (dict(into=torch.zeros((1, 2), dtype=I32)), "block tables"),
    (dict(into=torch.zeros((2, 2), dtype=torch.int64)), "into"),
    (dict(sums_out=torch.zeros(2, 3, 9)), "without sums"),
    (dict(sums=torch.zeros(2, 2, 9)), "sums"),
    (dict(sums=torch.zeros(2, 3, 9), sums_out=torch.zeros(2, 3, 9, dtype=torch.bfloat16)), "sums"),
])
def test_moving_refuses(no_launch, change, match):
    with pytest.raises(K.KernelError, match=match):
        K.kv_compact(**_compact(**change))


def test_sums_move_within_themselves_or_apart(no_launch):
    one = torch.zeros(100)
    with pytest.raises(K.KernelError, match="apart"):
        K.kv_compact(**_compact(sums=one[:54].view(2, 3, 9), sums_out=one[6:60].view(2, 3, 9)))
    with pytest.raises(K.KernelError, match="apart"):
        K.kv_compact(**_compact(sums=one[:54].view(2, 3, 9), sums_out=one[:48].view(2, 3, 8)))


@pytest.mark.parametrize("count, page, dh", [(0, 16, 64), (4, 0, 64), (4, 16, 0)])
def test_moving_refuses_pages_without_rows(no_launch, count, page, dh):
    with pytest.raises(K.KernelError, match="16 bytes"):
        K.kv_compact(**_compact(pages=torch.zeros(count, 2, 3, page, dh)))


def test_a_choice_writes_over_nothing_that_it_reads(no_launch, monkeypatch):
    """Heads of a request read its length and number while another one may have written its count already."""
    monkeypatch.setattr(K, "_placed", lambda *a: -1)  # as if the tensors were on the device
    a = _choose()
    many = torch.zeros(60, dtype=I32)
    for change in (dict(counts=a["lengths"], lengths=a["lengths"]), dict(counts=a["keep"], keep=a["keep"]), dict(lengths=many[:2], counts=many[1:3]),
                   dict(places=many[:24].view(2, 3, 4), counts=many[22:24]), dict(places=many[:24].view(2, 3, 4), lengths=many[10:12]),
                   dict(places=many[:24].view(2, 3, 4), keep=many[23:25]), dict(sums=many.view(torch.float32).view(2, 3, 10), places=many[:24].view(2, 3, 4)),
                   dict(sums=many.view(torch.float32).view(2, 3, 10), counts=many[58:])):
        with pytest.raises(K.KernelError, match="share memory"):
            K.kv_choose(**_choose(**change))
    # entries behind a request's are not used; places of no size lie nowhere
    ran = []
    monkeypatch.setattr(K, "_run", lambda *args: ran.append(args))
    monkeypatch.setattr(K, "_raw_stream", lambda dev: None)
    monkeypatch.setattr(K, "sm_count", lambda: 148)
    K.kv_choose(**_choose(lengths=many, keep=many[2:], counts=many[4:]))
    K.kv_choose(**_choose(lengths=many, keep=many[2:], counts=many[4:], places=many[:0].view(2, 3, 0)))
    assert len(ran) == 2


def test_the_width_of_the_sums_does_not_change_the_blocks_of_a_call(no_launch, monkeypatch):
    """Tiles of keys that a block has one after the other go by the keys that requests have, not by the places that `out` has room for."""
    ran = []
    monkeypatch.setattr(K, "_placed", lambda *a: 0)  # as if the tensors were on the device, and a launch a note of its arguments
    monkeypatch.setattr(K, "_raw_stream", lambda dev: None)
    monkeypatch.setattr(K, "sm_count", lambda: 148)
    monkeypatch.setattr(K, "_run", lambda lib, fn, args, more, *rest: ran.append(rest))
    for width in (4096, 8192, 600000):
        K.attention_weights(**_weights(out=torch.zeros(1, 2, width), max_kv_len=4096, max_count=64))
    assert ran[0] == ran[1] == ran[2] and ran[0][2] == 1
    # several where the keys themselves make more blocks than the device holds many times over
    K.attention_weights(**_weights(out=torch.zeros(1, 2, 200000), max_kv_len=200000, max_count=64))
    assert ran[3][2] > 1
