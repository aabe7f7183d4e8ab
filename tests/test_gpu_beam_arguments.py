"""Arguments of the operators of beam search as a caller may hand them over."""
from types import SimpleNamespace

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


def test_out_on_another_device_is_not_written():
    """Small calls go to the decode kernel only with arguments that both paths take."""
    import torch
    from fused_turboquant_b200 import PagedKVPool
    pool = PagedKVPool(8, 2, 128, 4, 4)
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 8, 128, dtype=torch.bfloat16, device="cuda")
    args = q, torch.zeros(2, 2, **i32), torch.full((2,), 20, **i32), 32, torch.tensor([16], **i32)

    def out_on(device):
        return SimpleNamespace(is_cuda=True, device=device, dtype=q.dtype, shape=q.shape, is_contiguous=lambda: True)

    assert not pool._takes_shared_kernel(*args, None, None)
    assert not pool._takes_shared_kernel(*args, out_on(q.device), None)
    assert pool._takes_shared_kernel(*args, out_on(torch.device("cuda", q.device.index + 1)), None)
