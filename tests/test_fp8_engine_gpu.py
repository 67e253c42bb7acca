"""An engine whose cache is kept in 8 bits, beside one that keeps the same rounded rows in bfloat16.

Both attend over the same numbers (what 8 bits hold is exact in bfloat16), so their logits differ by the rounding of bfloat16
activations alone, the bound that every bfloat16 run of these models is held to."""

import random

import pytest
import torch

from tests import helpers as H

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
MODELS = {
    64: dict(moe_layers=[]),
    128: dict(moe_layers=[], head_dim=128, hidden_size=256, num_attention_heads=4, num_key_value_heads=2),
}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("fp8_models")
    return {dh: H.make_model_dir(root / f"head{dh}", "tiny_c", seed=5, norm_noise=0.05, **over) for dh, over in MODELS.items()}


def _round_rows(monkeypatch):
    """Makes the bfloat16 engine write what 8 bits would hold of its keys and values."""
    from jax_llm_examples_b200.kernels import api as K

    def store(qkv, q_out, pages, block_table, req_of_token, positions, inv_freq, l2norm, eps, Hq, Hkv, dh, status, splits=1):
        n = q_out.shape[0]
        codes = torch.empty((n, 2, Hkv, 1, dh), dtype=FP8, device="cuda")  # a page of one token for every row of the step
        scales = torch.empty((n, 2, Hkv, 1), dtype=torch.uint8, device="cuda")
        own = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].contiguous()
        rows, zero = own.flatten().contiguous(), torch.zeros(n, dtype=torch.int32, device="cuda")
        K.rope_kv_store_fp8(qkv, q_out, codes, scales, own, rows, positions, inv_freq, l2norm, eps, Hq, Hkv, dh, status, splits, places=zero)
        k, v = (torch.empty((n, Hkv, dh), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        K.kv_load_fp8(codes, scales, own, rows, zero, k, v, status)
        K.kv_store(k, v, pages, block_table, req_of_token, positions, status)

    monkeypatch.setattr(K, "rope_kv_store", store)


def _trace(kind, reqs, seed):
    return {"whole": H.trace_whole, "tail": H.trace_tail_decode, "portions": lambda r: H.trace_portions(r, random.Random(seed)),
            "mixed": lambda r: H.trace_mixed(r, random.Random(seed), portions=H.LONG_PORTIONS)}[kind](reqs)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("kind, page", [("whole", 16), ("tail", 64), ("portions", 16), ("mixed", 64), ("mixed", 7)])
def test_the_engine_attends_over_what_8_bits_hold(folders, monkeypatch, dh, kind, page):
    import jax_llm_examples_b200 as J

    reqs = H.random_requests(random.Random(11), 320, [200, 81, 3, 260, 65, 129])
    model = J.load_model(folders[dh], "bfloat16")
    eight = J.Engine(model, max_tokens=900, page_size=page, max_slots=8, cache_dtype=FP8)
    got, _ = H.run_trace(eight, _trace(kind, reqs, 4), record_routing=False)
    assert kind != "tail" or eight.graph_replays > 0
    _round_rows(monkeypatch)
    plain = J.Engine(model, max_tokens=900, page_size=page, max_slots=8, use_graphs=False)
    want, _ = H.run_trace(plain, _trace(kind, reqs, 4), record_routing=False)
    worst = max(H.rel_err(got[k], want[k]) for k in want)
    assert got.keys() == want.keys() and worst < H.TOL["bfloat16"], worst
    assert all(eight.manager.free_pages(g) == eight.num_pages for g in range(len(eight.manager.groups)))


def test_the_cache_takes_half_the_memory_and_generation_runs_on_it(folders):
    import jax_llm_examples_b200 as J

    model = J.load_model(folders[128], "bfloat16")
    bf16 = J.Engine(model, max_tokens=640, page_size=16, max_slots=4)
    eight = J.Engine(model, max_tokens=640, page_size=16, max_slots=4, cache_dtype=FP8)
    assert eight.cache_bytes() * 256 == bf16.cache_bytes() * 129
    assert J.Engine.tokens_that_fit(model, 16, 0.5, FP8) > 1.9 * J.Engine.tokens_that_fit(model, 16, 0.5)
    prompts = [[7, 8, 9, 10] * 20, [5], [3, 1, 4, 1, 5, 9, 2, 6] * 9]
    params = J.SamplingParams(max_new_tokens=12)
    a = J.generate(model, prompts, params, page_size=16, cache_dtype=FP8)
    assert [len(x) for x in a] == [12] * 3
    assert a == J.generate(model, prompts, params, page_size=16, cache_dtype=FP8)


def test_models_that_take_no_8_bit_cache_are_refused(model_dirs, folders):
    import jax_llm_examples_b200 as J

    for folder, dtype in ((model_dirs["tiny_a"], "bfloat16"), (folders[64], "float32")):
        with pytest.raises(J.engine.EngineError, match="cannot be kept"):
            J.Engine(J.load_model(folder, dtype), max_tokens=64, page_size=16, max_slots=1, cache_dtype=FP8)
    with pytest.raises(J.engine.EngineError, match="cannot be kept"):
        J.Engine(J.random_model(J.preset("marinex_tiny"), 0), max_tokens=64, page_size=16, max_slots=1, cache_dtype=FP8)
