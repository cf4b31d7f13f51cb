"""Calls of the budget operators that are turned away before anything is launched, where sizes pass 32 bits or rows share memory."""
import pytest
import torch
from test_budget_cpu import B, BS, D, H, KV, N, T, _args, _call, on_the_cpu  # noqa: F401

from inference_b200.ops.runtime import KernelError


@pytest.mark.parametrize("name", ["selected", "tracked"])
@pytest.mark.parametrize("stride", [0, H * D - 1])
def test_results_whose_rows_share_memory_are_refused(name, stride):
    a = _args()
    a["out"] = torch.zeros(2 * H * D).bfloat16().as_strided((T, H * D), (stride, 1))
    with pytest.raises(KernelError, match="share"):
        _call(name, a)
    a["out"] = a["out"].as_strided((T, H * D), (H * D, 1))
    with pytest.raises(AssertionError, match="was launched"):
        _call(name, a)


@pytest.mark.parametrize("top,first,last", [(2 ** 31 - 1, 1, 4), (2 ** 31, 0, 1), (2 ** 30, 2 ** 30, 1), (1, 2 ** 31 - 2, 1), (1, 0, 2 ** 40)])
def test_selections_whose_width_passes_32_bits_are_refused(top, first, last):
    a = _args() | {"top": top, "first": first, "last": last}
    with pytest.raises(KernelError, match="2\\^31"):
        _call("select", a)


def test_the_library_refuses_a_selection_whose_width_passes_32_bits():
    """Whoever calls it: the check stands in front of the launch (the pointers are not read)."""
    from inference_b200._native import kernels
    from inference_b200.ops.budget import _INTS

    at = 1 << 20
    dims = _INTS[14](1, 1, 1, 8, 20, 4, KV, 2, D, 2 ** 30, 2 ** 30, 1, 0, 0)
    assert kernels().swb_page_select(dims, at, D, D, at, at, at, 8, None, at, at, at, None) == -3


@pytest.mark.parametrize("name,key", [("summaries", "max_q"), ("select", "max_q"), ("selected", "max_q"), ("tracked", "max_q"), ("select", "bs"), ("evict", "keep")])
def test_sizes_behind_32_bits_are_refused_as_arguments(name, key):
    a = _args() | {key: 2 ** 31}
    if key == "max_q":
        a["cu"] = torch.zeros(B + 1, dtype=torch.int32)
    with pytest.raises(KernelError):
        _call(name, a)


def test_the_library_refuses_summaries_of_a_table_for_2_to_the_31_tokens():
    """As it refuses such a table for the other operators: places in a sequence are 32-bit numbers. (The pointers are not read.)"""
    from inference_b200._native import kernels
    from inference_b200.ops.budget import _INTS

    at = 1 << 20
    assert kernels().swb_page_summaries(_INTS[9](1, 1, 2 ** 27, 20, 16, KV, D, 0, 0), at, at, at, at, 2 ** 27, None, at, None) == -3


def test_the_library_refuses_a_grid_of_more_than_2_to_the_31_blocks():
    """Tokens that share their keys are dealt out by the longest step a sequence may have, which can be many more blocks than there are tokens."""
    from inference_b200._native import kernels
    from inference_b200.ops.budget import _INTS, _LONGS

    at, seqs, most = 1 << 20, 65535, 2 ** 20
    dims = _INTS[16](8, seqs, most, 1, 20, 16, 1, 1, 128, 128, 0, 1, 0, 0, 0, 0)
    strides = _LONGS[8](128, 128, 128, 1, 16, 16, 0, 0)
    assert kernels().swb_attn_budget(dims, strides, at, at, at, at, at, at, at, None, None, at, 1.0, 0.0, at, 1 << 20, None) == -3


@pytest.mark.parametrize("max_seq_len,heads,kv_heads,width", [(16 * 40000 + 1, 8, 2, 64), (1024, 129, 1, 16), (1024, 8, 2, 264)])
def test_a_page_budget_that_no_step_could_keep_is_refused_with_its_runner(max_seq_len, heads, kv_heads, width):
    """Contexts of more pages than a selection is made over, more query heads to a key/value head and wider heads than its operators take: at once, not at the first step."""
    from inference_b200.contracts.errors import Unsupported
    from inference_b200.engine.kv_pool import PagedKvPool
    from inference_b200.engine.runner import ModelRunner
    from inference_b200.models.llama import LlamaGpu
    from inference_b200.ops import PageBudget

    model = LlamaGpu.__new__(LlamaGpu)
    model.hq, model.hkv = heads, kv_heads
    pool = PagedKvPool(1, 2, kv_heads, width, device="cpu")
    with pytest.raises(Unsupported):
        ModelRunner(model, pool, max_batch=1, max_seq_len=max_seq_len, page_budget=PageBudget(top=1))
    assert pool.summaries is None


@pytest.mark.parametrize("pages,weights", [(False, False), (True, True)])
def test_the_library_takes_page_lists_or_weights(pages, weights):
    from inference_b200._native import kernels
    from inference_b200.ops.budget import _INTS, _LONGS

    at = 1 << 20
    dims, strides = _INTS[16](1, 1, 1, 8, 20, 16, 1, 1, 128, 128, 3, 1, 0, 0, 0, 0), _LONGS[8](128, 128, 128, 8, 128, 128, 0, 0)
    assert kernels().swb_attn_budget(dims, strides, at, at, at, at, at, None, at, at if pages else None, at if pages else None, at if weights else None, 1.0, 0.0, at, 1 << 20,
                                     None) == -3
