"""beam.select on masked logits: what a mask rules out is never a candidate."""
import math

import pytest
from test_gpu_beam_select import check, random_case

pytestmark = pytest.mark.gpu
MASKED = 0x007fffff       # of a key's upper half: the order of -inf


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("left", [1, 5, 50, 3000])
@pytest.mark.parametrize("V", [4099, 70000])
def test_a_grammar_that_leaves_some_tokens(V, left, dtype):
    """The answer, and that no masked token takes the place of a candidate in the scratch memory."""
    import torch
    from fused_turboquant_b200 import beam
    x, s = random_case(3, 4, V, getattr(torch, dtype))
    g = torch.Generator("cuda").manual_seed(left)
    allowed = torch.rand(x.shape, device="cuda", generator=g).argsort(-1)[..., :left]
    y = torch.full_like(x, -math.inf).scatter_(-1, allowed, x.gather(-1, allowed))
    y[1, 2] = x[1, 2].sort().values                    # (a row without a mask, and one with a block of allowed tokens)
    y[2, 0, :] = -math.inf
    y[2, 0, 17:17 + left] = x[2, 0, 17:17 + left]
    ends = allowed[0, 0, :1]
    ws = torch.zeros(beam.workspace_bytes(x.dtype, 3, 4, V, 9, 1), dtype=torch.uint8, device="cuda")
    check(y, s, 9, ends=ends, workspace=ws)
    assert not ((ws.view(torch.int64) >> 32) == MASKED).any()


def test_a_mask_that_leaves_nothing():
    import torch
    x, s = random_case(2, 3, 50257, torch.float32)
    x[0] = -math.inf
    x[1, :2] = -math.inf
    got = check(x, s, 6)
    assert (got.tokens[0] == -1).all() and (got.parents[1] == 2).all()
