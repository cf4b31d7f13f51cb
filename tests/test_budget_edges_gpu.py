"""Operators of long caches on a budget where their definitions are easily missed: calls that the documentation allows and that differ from the usual ones."""
import pytest
import torch
from test_budget_gpu import CUDA, Cache, _ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("splits", [1, 3, 9])
def test_pages_that_are_not_there_weigh_nothing_beside_a_key_that_is_no_number(splits, kind):
    """However a problem's splits are joined and its weights added up."""
    ops = _ops()
    c = Cache([100], [1], kind=kind)
    c.k[c.table[0, 0].long(), 1, 5] = float("nan")
    c.table[0, 2] = -5
    weights = torch.zeros(1, 2, c.per * 16, device=CUDA)
    ops.tracked_attention(c.q, c.k, c.v, c.table, c.kv_lens, weights, scale=0.1, num_splits=splits, **c.step)
    there = torch.tensor([j // 16 != 2 for j in range(100)], device=CUDA)
    assert weights[0, 1, :100][there].isnan().all() and weights[0, 0].isfinite().all()
    assert weights[0, :, 32:48].eq(0).all() and weights[0, :, 100:].eq(0).all()
