"""What the operators of drafted trees, page copies and beams hand to the library, before anything is launched."""
import struct

import pytest
import torch

from inference_b200._native import kernels
from inference_b200.ops import branch
from inference_b200.ops.runtime import KernelError


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


@pytest.mark.parametrize("bs", [1, 16, 48])
def test_tables_whose_ends_pass_32_bits_are_refused(calls, bs):
    """Tiles reach behind a sequence's end: the last places of a table that is nearly 2^31 tokens long would be numbers below zero."""
    z, pages = torch.zeros, (2 ** 31 - 1) // bs

    def run(pages):
        return branch.tree_attention(z(1, 2, 16).bfloat16(), z(3, 1, bs, 16).bfloat16(), z(3, 1, bs, 16).bfloat16(), torch.empty((1, pages), dtype=torch.int32, device="meta"),
                                     z(1, dtype=torch.int32), z(1, 1, dtype=torch.int32), cu_q=None, max_q_len=1, scale=1.0)

    with pytest.raises(KernelError):
        run(pages)
    assert not calls
    run((2 ** 31 - 1025) // bs)
    assert "swb_attn_tree" in calls
    # and by the library, in front of every launch
    dims = struct.pack("16i", 1, 1, 1, pages, 3, bs, 1, 2, 16, 16, 1, 1, 0, 0, 0, 0)
    assert kernels().swb_attn_tree(dims, struct.pack("8q", 32, 16, 32, pages, 1, 0, 0, 0), 16, 16, 16, 16, 16, None, 16, 16, 1.0, 0.0, None, 0, None) == -3
