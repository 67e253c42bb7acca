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
