"""What the operators of drafted trees, page copies and beams hand to the library, before anything is launched."""
import struct

import pytest
import torch

from inference_b200.ops import branch


class _Calls:
    """Takes down the calls of the library's functions."""

    def __init__(self):
        self.made = {}

    def __getattr__(self, name):
        def call(*args):
            self.made[name] = args
            return 0
        return call


@pytest.fixture
def calls(monkeypatch):
    made = _Calls()
    monkeypatch.setattr(branch, "kernels", lambda: made)
    monkeypatch.setattr(branch, "_place", lambda *a: 0)
    return made.made


@pytest.mark.parametrize("bound", [40, 4096, 2 ** 31 - 1])
def test_a_steps_bound_may_be_far_above_its_tokens(calls, bound):
    """Masks are as wide as the step has tokens, and no more row tiles are launched."""
    z = torch.zeros
    cu, T = torch.tensor([0, 33, 40], dtype=torch.int32), 40
    plan = branch.plan_tree(z(T, dtype=torch.int32), cu_q=cu, max_q_len=bound)
    assert plan.mask.shape == (T, 2) and calls["swb_plan_tree"][3] == T
    out = branch.tree_attention(z(T, 4, 16).bfloat16(), z(20, 2, 16, 16).bfloat16(), z(20, 2, 16, 16).bfloat16(), z(2, 8, dtype=torch.int32), z(2, dtype=torch.int32), plan.mask,
                                cu_q=cu, max_q_len=bound, scale=1.0)
    dims = struct.unpack("16i", calls["swb_attn_tree"][0])
    assert out.shape == (T, 64) and dims[:3] == (T, 2, T) and dims[11] == branch.tree_splits(2 * 2 * 1, 8 * 16)
