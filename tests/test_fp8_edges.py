"""The 8-bit cache and the attention over rows, where their format, their plans and their calls end: what needs no GPU."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "jax_llm_examples_b200" / "csrc"


def _code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


@pytest.mark.parametrize("name, stores, release", [
    ("attention_few.cu", "*at = make_uint4(0u, 0u, 0u, 0u);", "mbar_arrive(EMPTY(st))"),
    ("attention_rows_tc.cu", "*at = make_uint4(w[0], w[1], w[2], w[3]);", "mbar_arrive(BAR(B_VREADY + st))"),
])
def test_values_changed_in_a_stage_are_fenced_before_it_is_filled_again(name, stores, release):
    """Ordinary stores into a stage that TMA fills next: the lanes that stored have to order them before the asynchronous proxy's
    writes (a missing fence shows on no test's numbers, only in the order that the memory model grants)."""
    code = _code(name)
    at = code.index(stores)
    between = code[at:code.index(release, at)]
    assert "fence.proxy.async" in between or "fence_async_proxy()" in between


def test_the_largest_row_that_is_held_is_448_times_2_to_the_60():
    """The kernels' limit is the format's: 448 * 2^60, to the last bit of a 32-bit number."""
    import numpy as np

    text = re.search(r"#define FP8_LIMIT (\S+?)f\s", (CSRC / "fp8_rows.cuh").read_text() + "\n").group(1)
    value = float.fromhex(text) if text.lower().startswith("0x") else float(text)
    assert np.float32(value) == np.float32(448 * 2.0 ** 60)


# (kept heads, rows of a step, its items or single rows, keys of the longest request)
SCRATCH = [
    # one decoded token behind a long context beside a prompt's portion
    (40, 8, 128, 2049, dict(rows=1), 30000), (40, 8, 128, 8193, dict(rows=1), 131072), (16, 2, 64, 2050, dict(rows=2), 131072),
    # short portions beside a long one, and drafted trees of one request out of many tokens
    (40, 8, 128, 2100, dict(items=3, most=16), 30000), (32, 8, 128, 5000, dict(items=1, most=64), 131072),
    # one list of portions of very different lengths, sized by the longest
    (40, 8, 128, 2250, dict(items=101, most=2048), 30000),
    # portions of many rows a KV head, whole
    (64, 1, 128, 8192, dict(items=1, most=8192), 131072), (64, 1, 64, 16384, dict(items=1, most=16384), 131072), (40, 8, 128, 8192, dict(items=64, most=128), 8192),
]


@pytest.mark.parametrize("page", [64, 24])
@pytest.mark.parametrize("Hq, Hkv, dh, N, served, keys", SCRATCH)
def test_scratch_for_ranges_is_sized_by_the_rows_that_a_call_serves_and_bounded(monkeypatch, Hq, Hkv, dh, N, served, keys, page):
    import torch

    from jax_llm_examples_b200.kernels import api as K

    asked, ran = [], []
    monkeypatch.setattr(K, "_placed", lambda *a: 0)
    monkeypatch.setattr(K, "_raw_stream", lambda dev: None)
    monkeypatch.setattr(K, "sm_count", lambda: 148)
    monkeypatch.setattr(K, "_few_places", lambda *a: (444,) * len(K.ROWS_SPLITS))
    monkeypatch.setattr(K, "_run", lambda lib, fn, args, stream: ran.append(K._ROWS_ARGS.unpack(args)))
    q = torch.zeros((N, Hq, dh), dtype=torch.bfloat16)
    pages = torch.zeros((2, 2, Hkv, page, dh), dtype=torch.uint8).view(K.FP8)
    ints = torch.zeros(N, dtype=torch.int32)
    items, most = served.get("items", 0), served.get("most", 1)
    out, pairs = torch.empty_like(q), torch.zeros((items, 2), dtype=torch.int32) if items else None
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda n, **kw: asked.append(n * 4) or empty(0, **kw))
    K.attention_fp8(q, pages, torch.zeros((2, 2, Hkv, page), dtype=torch.uint8), torch.zeros((1, 2), dtype=torch.int32), ints, ints, out, 1.0, 0, 0, 0.0, 1.0,
                    torch.zeros(1, dtype=torch.int32), keys, items=pairs, n_items=items, max_count=most, rows=ints if "rows" in served else None,
                    n_rows=served.get("rows", 0))
    assert len(ran) == 1
    rows = min(N, served["rows"] if "rows" in served else items * most)
    for n in asked:
        assert n <= 256 << 20 and n <= rows * Hq * max(K.ROWS_SPLITS) * (dh + 2) * 4


def _attend_args(**change):
    import torch

    from .fp8_helpers import Case

    c = Case([3], [5], 4, 2, 64, 16, device="cpu")
    a = dict(q=c.q, pages=c.pages, scales=c.scales, block_table=c.table, req_of_token=c.req, positions=c.positions, out=torch.empty_like(c.q),
             scale=0.125, chunk=0, window=0, attn_scale=0.0, floor_scale=1.0, status=c.status, max_kv_len=8)
    return {**a, **change}


def test_items_and_single_rows_in_one_call_are_refused(monkeypatch):
    """One of the two would be left out of the output, and the caller not told."""
    import torch

    from jax_llm_examples_b200.kernels import api as K

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(K.KernelError, match="items or single rows"):
        K.attention_fp8(**_attend_args(items=torch.zeros((1, 2), dtype=torch.int32), n_items=1, max_count=3, rows=torch.zeros(1, dtype=torch.int32), n_rows=1))


def test_an_output_that_shares_memory_with_the_queries_is_refused(monkeypatch):
    """Blocks read queries while others write outputs."""
    import torch

    from jax_llm_examples_b200.kernels import api as K

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    room = torch.zeros(5 * 4 * 64, dtype=torch.bfloat16)
    q = room[:3 * 256].view(3, 4, 64)
    for first in (0, 1, 2):
        with pytest.raises(K.KernelError, match="not the same rows"):
            K.attention_fp8(**_attend_args(q=q, out=room[first * 256:(first + 3) * 256].view(3, 4, 64)))


def test_what_two_8_bit_parts_hold_of_a_query():
    """An e4m3 part and what is left of it in e5m2, of every bfloat16 number up to 2^8: exact from 2^-6 on, off by 2^-14 at most below."""
    import torch

    a = torch.arange(0x7F80, dtype=torch.int16).view(torch.bfloat16).float()
    a = a[a < 256]
    first = a.to(torch.float8_e4m3fn).float()
    off = (a.double() - first.double() - (a - first).to(torch.float8_e5m2).double()).abs()
    assert not off[a >= 2.0 ** -6].any() and off.max() == 2.0 ** -14
