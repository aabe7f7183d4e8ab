"""beam.select where beams say the same: equal totals go to the lowest beam, wherever the rows lie in memory."""
import math

import pytest
from test_gpu_beam_select import check, random_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("K,V,n", [(8, 50257, 24), (3, 4099, 64), (2, 300001, 9), (64, 1001, 64), (5, 9, 30)])
def test_beams_that_say_the_same(K, V, n, dtype):
    """Rows of an odd length begin at every place between two 16-byte boundaries."""
    import torch
    x, _ = random_case(3, K, V, getattr(torch, dtype))
    x[:] = x[:, :1].clone()
    s = torch.zeros(3, K, device="cuda")
    s[1] = -7.3
    got = check(x, s, n, ends=torch.tensor([V // 2], device="cuda"))
    assert got.scores[0, :min(K, n)].unique().numel() == 1 and got.parents[0, :min(K, n)].tolist() == list(range(min(K, n)))
    s[2, ::2] = -math.inf
    check(x, s, n)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("V", [5, 513, 4099, 70000, 131072])
def test_rows_at_any_place_give_the_same_bits(V, dtype):
    import torch
    from fused_turboquant_b200 import beam
    x, s = random_case(2, 3, V, getattr(torch, dtype))
    want = check(x, s, 20)
    for at in range(16 // x.element_size()):
        for gap in (16, 17):
            base = torch.full((2, 3, V + gap), 100.0, dtype=x.dtype, device="cuda")
            base[..., at:at + V] = x
            got = beam.select(base[..., at:at + V], s, 20)
            assert all(torch.equal(a, b) for a, b in zip(got[:3], want[:3]))
