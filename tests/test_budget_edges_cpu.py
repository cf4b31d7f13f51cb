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
