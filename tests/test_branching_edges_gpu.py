"""Drafted trees, beams and page copies through the engine on the GPU, where their calls are easily missed."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_page_that_is_copied_to_itself_stays():
    from inference_b200.engine.kv_pool import KvGeometry, LayeredKvPool, PagedKvPool

    pool = PagedKvPool(2, 5, 1, 64, 16)
    pool.data.copy_(torch.randn(pool.data.shape))
    want = pool.data.clone()
    pool.copy_block(3, 3)
    assert torch.equal(pool.data, want)
    pool.copy_blocks([1, 2, 1], [1, 4, 0])
    want[:, :, [4, 0]] = want[:, :, [2, 1]]
    assert torch.equal(pool.data, want)
    layered = LayeredKvPool([KvGeometry(1, 8, 8)], 3, 16)
    layered.copy_block(1, 1)
    layered.copy_state(0, 1)        # it keeps none
