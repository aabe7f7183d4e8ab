"""beam.select against the definition in 64 bits."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def plain(logits, scores, n, ends=None):
    """(scores, parents, tokens, end scores) of the definition, in 64 bits."""
    import torch
    x = logits.double().cpu()
    R, K, V = x.shape
    total = torch.log_softmax(x, -1) + scores.double().cpu()[..., None]
    total = torch.where(torch.isnan(total), -math.inf, total)
    end_scores = None
    if ends is not None:
        ok = (ends >= 0) & (ends < V)
        end_scores = torch.where(ok, total[..., ends.clamp(0, V - 1).long()], -math.inf)
        total[..., ends[ok].long()] = -math.inf
    flat, order = total.view(R, -1).sort(dim=-1, descending=True, stable=True)
    flat, order = flat[:, :n], order[:, :n]
    pad = n - flat.shape[1]
    flat, order = torch.nn.functional.pad(flat, (0, pad), value=-math.inf), torch.nn.functional.pad(order, (0, pad))
    none = flat == -math.inf
    return flat, torch.where(none, -1, order // V), torch.where(none, -1, order % V), end_scores


def close(got, want, V):
    """A total is the score, a logit and a log sum exp, rounded once: half a step of fp32 of the total, and of the sum what its parts
    add: exp's argument is rounded (2^-24 of up to |x| log2 e, where the weight 2^-|x| makes at most 2^-24 of it) and exp2 itself is good to
    2^-22; a thread adds up to 32 * 32 terms in 4 chains, then 9 sums: at most 300 roundings of 2^-24.  Together under 2^-15."""
    import torch
    got, want = got.double().cpu(), want.double()
    assert torch.equal(torch.isfinite(got), torch.isfinite(want))
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine], want[~fine])
    assert ((got - want)[fine].abs() <= 2.0 ** -24 * want[fine].abs() + 2.0 ** -15).all()


def check(logits, scores, n, ends=None, **kw):
    import torch
    from fused_turboquant_b200 import beam
    got = beam.select(logits, scores, n, end_tokens=ends, **kw)
    s, p, t, e = plain(logits, scores, n, None if ends is None else ends.cpu())
    assert got.parents.dtype == got.tokens.dtype == torch.int32 and got.scores.dtype == torch.float32
    assert torch.equal(got.parents.cpu().long(), p)
    assert torch.equal(got.tokens.cpu().long(), t)
    close(got.scores, s, logits.shape[-1])
    if ends is None:
        assert got.end_scores is None
    else:
        close(got.end_scores, e, logits.shape[-1])
    return got


def random_case(R, K, V, dtype, seed=0, scale=2.5):
    import torch
    g = torch.Generator("cuda").manual_seed(seed + V)
    x = (scale * torch.randn(R, K, V, device="cuda", generator=g)).to(dtype)
    return x, -5 * torch.rand(R, K, device="cuda", generator=g)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("R,K,V,n", [
    (1, 1, 1, 1), (1, 1, 2, 4), (2, 3, 7, 5), (1, 4, 8, 64), (3, 2, 513, 9), (1, 4, 32768, 4), (2, 5, 50257, 10), (1, 64, 999, 64),
    (70, 8, 4099, 16), (2, 1, 300001, 3), (160, 2, 131072, 2), (1, 1, 65536 * 5 + 3, 33), (400, 1, 1000, 1)])
def test_sizes(R, K, V, n, dtype):
    import torch
    x, s = random_case(R, K, V, getattr(torch, dtype))
    check(x, s, n)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("R,K,V,n,ends", [(3, 4, 1000, 4, [0]), (2, 8, 40000, 16, [39999, 5, 17, 17]), (1, 64, 200, 64, list(range(0, 160, 10))),
                                          (2, 2, 10, 3, [-1, 10, 3, 2 ** 31 - 1]), (1, 3, 5, 8, [0, 1, 2, 3, 4])])
def test_tokens_that_end_an_answer(R, K, V, n, ends, dtype):
    """The likeliest tokens too; ids outside the vocabulary have no total."""
    import torch
    x, s = random_case(R, K, V, getattr(torch, dtype))
    e = torch.tensor(ends, device="cuda")
    ok = e[(e >= 0) & (e < V)]
    x[..., ok[: max(1, len(ok) // 2)]] += 20
    check(x, s, n, ends=e)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("V", [5, 3000, 70000, 131072])
def test_ties_go_to_the_lowest_place(V, dtype):
    """All logits equal; a few values only; ascending and descending rows; beams that say the same; zeros of both signs."""
    import torch
    t = getattr(torch, dtype)
    x = torch.zeros(2, 3, V, dtype=t, device="cuda")
    x[0, :, ::2] = -0.0
    check(x, torch.zeros(2, 3, device="cuda"), 12)
    g = torch.Generator("cuda").manual_seed(V)
    x = torch.randint(0, 3, (2, 4, V), device="cuda", generator=g).to(t)
    x[:, 1] = x[:, 0]
    check(x, torch.zeros(2, 4, device="cuda"), 40, ends=torch.tensor([1, 2], device="cuda"))
    up = torch.arange(V, device="cuda").float() / V
    check(torch.stack([up, up.flip(0)])[None].to(t), torch.tensor([[0.0, -0.01]], device="cuda"), 30)


def test_beams_that_are_not_alive():
    """The first step: one beam of each request; no beam at all; scores that are no numbers.  Dead rows are not looked at."""
    import torch
    x, s = random_case(4, 5, 3001, torch.bfloat16)
    s[:, 1:] = -math.inf
    s[2] = -math.inf
    s[3, 0] = math.nan
    x[0, 3] = math.nan
    x[1, 2] = math.inf
    got = check(x, s, 7, ends=torch.tensor([3], device="cuda"))
    assert (got.tokens[2:] == -1).all() and (got.scores[2:] == -math.inf).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits_that_are_no_numbers(dtype):
    import torch
    x, s = random_case(1, 6, 20001, getattr(torch, dtype))
    x[0, 0, 777] = math.nan
    x[0, 1, 20000] = math.inf
    x[0, 2] = -math.inf
    x[0, 3, 1:] = -math.inf           # a grammar that leaves one token
    x[0, 4, ::2] = -math.inf
    x[0, 5] = math.nan
    got = check(x, s, 9, ends=torch.tensor([0, 777], device="cuda"))
    assert set(got.parents[0].tolist()) <= {3, 4}
    x[0, 4] = -math.inf
    check(x, s, 9)                    # one token is left


def test_logits_of_very_different_size():
    import torch
    x, s = random_case(2, 3, 5000, torch.float32, scale=1.0)
    x[0, 0] *= 1e30
    x[0, 1] += 1e4
    x[0, 2] -= 3e38
    x[1, 0, 5] = -3e38
    s[1, 1] = -1e5
    check(x, s, 6)


def test_strides_and_places():
    """Rows apart, rows that begin anywhere, a transposed tensor."""
    import torch
    for dtype in (torch.bfloat16, torch.float32):
        base, s = random_case(3, 4, 5013, dtype)
        check(base[..., 3:4100], s, 8)
        check(base[..., 1:], s, 8)
        check(base.transpose(0, 1), s.T.contiguous(), 8)
        check(base[:, 1:3, 7:900], s[:, 1:3], 8)
        check(base[:, :, ::2], s, 8)
        check(base, s.double(), 8)


def test_an_empty_batch():
    import torch
    from fused_turboquant_b200 import beam
    got = beam.select(torch.empty(0, 4, 100, device="cuda"), torch.empty(0, 4, device="cuda"), 4, end_tokens=torch.tensor([1], device="cuda"))
    assert got.tokens.shape == (0, 4) and got.end_scores.shape == (0, 4, 1)


def test_logits_of_more_than_four_gigabytes():
    """Rows whose bytes lie beyond 32 bits."""
    import torch
    from fused_turboquant_b200 import beam
    x = torch.zeros(260, 64, 131072, dtype=torch.bfloat16, device="cuda")       # 4.4 GB
    x[259, 63, 131071] = 5
    s = torch.zeros(260, 64, device="cuda")
    got = beam.select(x, s, 2)
    assert got.parents[259].tolist() == [63, 0] and got.tokens[259].tolist() == [131071, 0]
    assert got.parents[258].tolist() == [0, 0] and got.tokens[258].tolist() == [0, 1]


def test_refusals():
    import torch
    from fused_turboquant_b200 import beam
    x, s = torch.zeros(2, 3, 10, device="cuda"), torch.zeros(2, 3, device="cuda")
    with pytest.raises(RuntimeError, match="CUDA"):
        beam.select(x.cpu(), s, 2)
    for bad in (x[0], x.double(), x.int()):
        with pytest.raises(ValueError, match="logits"):
            beam.select(bad, s, 2)
    with pytest.raises(ValueError, match="scores"):
        beam.select(x, s[:, :2], 2)
    for n in (0, -1, 65):
        with pytest.raises(ValueError, match="1 to 64"):
            beam.select(x, s, n)
    with pytest.raises(ValueError, match="1 to 64"):
        beam.select(torch.zeros(1, 65, 10, device="cuda"), torch.zeros(1, 65, device="cuda"), 2)
    with pytest.raises(ValueError, match="end_tokens"):
        beam.select(x, s, 2, end_tokens=torch.zeros(17, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="end_tokens"):
        beam.select(x, s, 2, end_tokens=torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="vocab"):
        beam.select(x[..., :0], s, 2)
    with pytest.raises(RuntimeError, match="workspace needs"):
        beam.select(x, s, 2, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


def test_captured_replayed_and_on_another_stream():
    import torch
    from fused_turboquant_b200 import beam
    x, s = random_case(3, 4, 9001, torch.bfloat16)
    ws = torch.empty(beam.workspace_bytes(x.dtype, 3, 4, 9001, 5, 1), dtype=torch.uint8, device="cuda")
    e = torch.tensor([9], dtype=torch.int32, device="cuda")
    beam.select(x, s, 5, end_tokens=e, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = beam.select(x, s, 5, end_tokens=e, workspace=ws)
    for seed in range(3):
        y, t = random_case(3, 4, 9001, torch.bfloat16, seed=50 + seed)
        x.copy_(y)
        s.copy_(t)
        graph.replay()
        want = plain(x, s, 5, e.cpu())
        assert torch.equal(got.tokens.cpu().long(), want[2]) and torch.equal(got.parents.cpu().long(), want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = beam.select(x, s, 5, end_tokens=e)
    side.synchronize()
    assert torch.equal(other.tokens, got.tokens) and torch.equal(other.scores, got.scores)


def test_the_same_call_gives_the_same_bits():
    import torch
    from fused_turboquant_b200 import beam
    x, s = random_case(20, 8, 32000, torch.bfloat16)
    first = beam.select(x, s, 16)
    for _ in range(5):
        again = beam.select(x, s, 16)
        assert all(torch.equal(a, b) for a, b in zip(first[:3], again[:3]))
