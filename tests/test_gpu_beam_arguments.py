"""Arguments of the operators of beam search as a caller may hand them over."""
import pytest

pytestmark = pytest.mark.gpu


def test_copies_that_32_bits_do_not_hold_are_outside_the_pool():
    import torch
    from fused_turboquant_b200 import PagedKVPool
    pool = PagedKVPool(8, 2, 64, 4, 4, n_layers=2)
    pool.pool.copy_(torch.randint(0, 256, pool.pool.shape, dtype=torch.uint8, device="cuda"))
    want = pool.pool.clone()
    want[:, 5] = want[:, 2]
    copies = [[1, (1 << 32) + 3], [(1 << 32) + 4, 6], [2, 5], [-(1 << 32), 7], [1 << 40, 0]]
    pool.copy_pages(torch.tensor(copies, device="cuda"))
    assert torch.equal(pool.pool, want)
