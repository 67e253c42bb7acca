"""The 8-bit cache's host side: the oracle against the format's table, refusals before anything is launched, tree masks."""

import math

import pytest
import torch

from jax_llm_examples_b200.kernels import api as K

from .fp8_helpers import Case, e4m3, hold


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


def test_the_oracles_grid_is_the_types_own():
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    grid = torch.unique(table[torch.isfinite(table)]).double()
    assert torch.equal(e4m3(grid), grid)
    between = (grid[1:] + grid[:-1]) / 2
    for x in (between, between + 1e-9, between - 1e-9, grid * 0.999):
        assert torch.equal(e4m3(x), x.float().to(torch.float8_e4m3fn).double() if torch.equal(x.float().double(), x) else grid[(x[:, None] - grid).abs().argmin(1)])


def test_a_rows_scale_is_the_smallest_that_holds_it():
    x = torch.tensor([[448.0, 1.0], [448.5, 1.0], [0.0, 0.0], [2.0 ** -80, 0.0], [3.5, -3.5000001], [math.inf, 1.0], [1.0, math.nan],
                      [448 * 2.0 ** 60, 0.0], [449 * 2.0 ** 60, 0.0]], dtype=torch.float64)
    _, s = hold(x)
    assert s.tolist() == [127, 128, 67, 67, 121, 255, 255, 187, 255]


def test_tree_masks():
    depth, bits = K.tree_masks([-1, 0, 0, 1, -1, 4])
    assert depth == [0, 1, 1, 2, 0, 1] and [b[0] for b in bits] == [1, 3, 5, 11, 16, 48]
    depth, bits = K.tree_masks(list(range(-1, 33)))  # a chain across two words, the sign bit among them
    assert depth[33] == 33 and bits[31] == [-1, 0] and bits[33] == [-1, 3]
    assert K.tree_masks([]) == ([], [])
    for bad in ([0], [-1, 1], [-1, -2]):
        with pytest.raises(K.KernelError, match="parent"):
            K.tree_masks(bad)


def _store_args(**change):
    c = Case([3], [5], 4, 2, 64, 16, device="cpu")
    a = dict(k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), pages=c.pages, scales=c.scales, block_table=c.table, req_of_token=c.req, places=c.places,
             status=c.status)
    return {**a, **change}


@pytest.mark.parametrize("change, match", [
    (dict(pages=torch.zeros(4, 2, 2, 16, 64)), "float8"),
    (dict(scales=torch.zeros(4, 2, 2, 16)), "uint8"),
    (dict(scales=torch.zeros((3, 2, 2, 16), dtype=torch.uint8)), "scales"),
    (dict(k=torch.zeros(3, 1, 64), v=torch.zeros(3, 1, 64)), "pages"),
    (dict(v=torch.zeros(3, 2, 64, dtype=torch.bfloat16)), "type"),
    (dict(k=torch.zeros(3, 64, 2).transpose(1, 2)), "contiguous"),
    (dict(places=torch.zeros(3)), "places"),
    (dict(places=torch.zeros(2, dtype=torch.int32)), "places"),
    (dict(req_of_token=torch.zeros(3, dtype=torch.int64)), "req_of_token"),
    (dict(block_table=torch.zeros((1, 2), dtype=torch.int64)), "block table"),
])
def test_store_and_load_refuse(no_launch, change, match):
    a = _store_args(**change)
    with pytest.raises(K.KernelError, match=match):
        K.kv_store_fp8(**a)
    with pytest.raises(K.KernelError, match=match):
        K.kv_load_fp8(a["pages"], a["scales"], a["block_table"], a["req_of_token"], a["places"], a["k"], a["v"], a["status"])


@pytest.mark.parametrize("change, match", [
    (dict(q=torch.zeros(3, 4, 64)), "bfloat16"),
    (dict(out=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), "bfloat16"),
    (dict(scales=None), "scales"),
    (dict(pages=torch.zeros((6, 2, 2, 16, 64), dtype=torch.bfloat16)), "float8"),
    (dict(max_kv_len=0), "keys"),
    (dict(items=torch.zeros((1, 2), dtype=torch.int32), n_items=2), "items"),
    (dict(items=torch.zeros((1, 2), dtype=torch.int32), n_items=1, max_count=0), "items"),
    (dict(rows=torch.zeros(1, dtype=torch.int32), n_rows=3), "rows"),
    (dict(sink=torch.zeros(3)), "sink"),
    (dict(slopes=torch.zeros(4, dtype=torch.float64)), "slopes"),
    (dict(positions=torch.zeros(3)), "positions"),
])
def test_attention_fp8_refuses(no_launch, change, match):
    c = Case([3], [5], 4, 2, 64, 16, device="cpu")
    a = dict(q=c.q, pages=c.pages, scales=c.scales, block_table=c.table, req_of_token=c.req, positions=c.positions, out=torch.empty_like(c.q),
             scale=0.125, chunk=0, window=0, attn_scale=0.0, floor_scale=1.0, status=c.status, max_kv_len=8)
    with pytest.raises(K.KernelError, match=match):
        K.attention_fp8(**{**a, **change})


@pytest.mark.parametrize("change, match", [
    (dict(masks=torch.zeros((2, 1), dtype=torch.int32)), "masks"),
    (dict(masks=torch.zeros(3, dtype=torch.int32)), "masks"),
    (dict(masks=None), "masks"),
    (dict(cu_q=torch.zeros(1, dtype=torch.int32)), "cu_q"),
    (dict(q_start=torch.zeros(1)), "q_start"),
    (dict(items=None), "items"),
    (dict(scales=None), "bfloat16"),
])
def test_attention_tree_refuses(no_launch, change, match):
    c = Case([3], [5], 4, 2, 64, 16, device="cpu").tree()
    a = dict(q=c.q, pages=c.pages, block_table=c.table, req_of_token=c.req, positions=c.positions, cu_q=c.cu_q, q_start=c.q_start, masks=c.masks,
             out=torch.empty_like(c.q), scale=0.125, chunk=0, window=0, attn_scale=0.0, floor_scale=1.0, status=c.status, max_kv_len=8,
             items=torch.tensor([[0, 3]], dtype=torch.int32), n_items=1, max_count=3, scales=c.scales)
    with pytest.raises(K.KernelError, match=match):
        K.attention_tree(**{**a, **change})


def test_tensors_that_are_not_on_the_gpu_are_refused(no_launch):
    with pytest.raises(K.KernelError, match="not on the GPU"):
        K.kv_store_fp8(**_store_args())


def test_an_engine_keeps_8_bits_only_where_every_layer_takes_them():
    from types import SimpleNamespace

    import jax_llm_examples_b200 as J
    from jax_llm_examples_b200.engine.engine import EngineError
    from jax_llm_examples_b200.parts.attention import GatedPagedAttention, PagedAttention
    from jax_llm_examples_b200.parts.base import Runtime
    from jax_llm_examples_b200.parts.positions import NoPositionWithTemperature, UnfusedEncoding

    bf16, f32 = (Runtime(t, torch.device("cpu")) for t in (torch.bfloat16, torch.float32))

    def mixer(dh, position, cls=PagedAttention):
        return PagedAttention(torch.zeros(4 * dh, 64), torch.zeros(64, 2 * dh), 2, 1, dh, position) if cls is PagedAttention else \
            GatedPagedAttention(torch.zeros(4 * dh, 64), torch.zeros(64, 2 * dh), 2, 1, dh, dh, 1.0, 1e-5, gate="none")

    fused = NoPositionWithTemperature()
    assert mixer(64, fused).takes_cache(K.FP8, bf16) and mixer(128, fused).takes_cache(K.FP8, bf16)
    assert not mixer(32, fused).takes_cache(K.FP8, bf16) and not mixer(64, fused).takes_cache(K.FP8, f32)
    assert not mixer(64, UnfusedEncoding()).takes_cache(K.FP8, bf16) and not mixer(64, None, GatedPagedAttention).takes_cache(K.FP8, bf16)
    assert mixer(32, fused).takes_cache(torch.bfloat16, bf16) and not mixer(32, fused).takes_cache(torch.float16, bf16)
    model = SimpleNamespace(runtime=bf16, takes_cache=lambda t: False)
    assert J.Engine.cache_type(model, None) == J.Engine.cache_type(model, torch.bfloat16) == torch.bfloat16
    for t in (K.FP8, torch.float16, torch.float32):
        with pytest.raises(EngineError, match="cannot be kept"):
            J.Engine.cache_type(model, t)
    model.takes_cache = lambda t: True
    assert J.Engine.cache_type(model, K.FP8) == K.FP8
    with pytest.raises(EngineError, match="cannot be kept"):
        J.Engine.cache_type(model, torch.float8_e5m2)
