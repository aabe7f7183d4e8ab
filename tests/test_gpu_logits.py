"""logits.process against its definition: bit for bit in fp32, and within its five roundings in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def plain(x, real, r, t, hist=None, hl=None, pl=None, rep=None, freq=None, pres=None, ids=None, bias=None, allowed=None, toks=None, masks=None):
    """The definition in the type `real`, and per value the largest magnitude that its steps pass through."""
    v = x.shape[-1]
    y = x.reshape(r, t, v).astype(real).copy()
    size = np.abs(y.astype(np.float64))
    for i in range(r):
        n, p = (min(int(hl[i]), hist.shape[1]), int(pl[i]) if pl is not None else 0) if hist is not None else (0, 0)
        prompt = hist[i, :min(p, n)] if hist is not None else []
        answer = hist[i, max(p, 0):n] if hist is not None else []
        for j in range(t):
            count = np.zeros(v, np.int64)
            more = [toks[i, k] for k in range(t) if masks[i, j, k // 32] >> (k % 32) & 1] if toks is not None else []
            for k in [*answer, *more]:
                if 0 <= k < v:
                    count[k] += 1
            seen = count > 0
            for k in prompt:
                if 0 <= k < v:
                    seen[k] = True
            a = y[i, j]
            if rep is not None:
                q = real(rep[i])
                a = np.where(seen, np.where(a > 0, a / q, a * q), a).astype(real)
            size[i, j] = np.maximum(size[i, j], np.abs(a))
            for pen, c in ((freq, count), (pres, count > 0)):
                if pen is not None:
                    step = (real(pen[i]) * c.astype(real)).astype(real)
                    a = np.where(count > 0, a - step, a).astype(real)
                    size[i, j] = np.maximum(size[i, j], np.maximum(np.abs(a), np.abs(step)))
            if ids is not None:
                for k, b in dict(zip(ids[i].tolist(), bias[i])).items():
                    if 0 <= k < v:
                        a[k] = a[k] + real(b)
                        size[i, j, k] = max(size[i, j, k], abs(a[k]))
            if allowed is not None:
                bits = np.unpackbits(allowed[i, j].view(np.uint8), bitorder="little")[:v]
                a = np.where(bits, a, -np.inf).astype(real)
            y[i, j] = a
    return y.reshape(x.shape), size.reshape(x.shape)


def make(rng, r, t, v, h=0, k=0, grammar=False, tree=False, penal=True):
    a = dict(r=r, t=t)
    if h:
        a["hist"] = rng.integers(0, max(1, min(v, 60)), (r, h)).astype(np.int32)
        a["hist"][rng.random((r, h)) < 0.02] = -1
        a["hist"][rng.random((r, h)) < 0.02] = v
        a["hist"][rng.random((r, h)) < 0.3] = rng.integers(0, v)
        a["hl"] = rng.integers(0, h + 1, r).astype(np.int32)
        a["hl"][0] = h
        a["pl"] = (a["hl"] * rng.random(r)).astype(np.int32)
    if penal:
        a.update(rep=rng.uniform(0.7, 1.6, r).astype(np.float32), freq=rng.uniform(-1, 1, r).astype(np.float32),
                 pres=rng.uniform(-1, 1, r).astype(np.float32))
    if k:
        a["ids"] = rng.integers(-1, v + 1, (r, k)).astype(np.int32)       # (some outside, some twice)
        a["bias"] = rng.normal(0, 5, (r, k)).astype(np.float32)
    if grammar:
        a["allowed"] = rng.integers(0, 1 << 32, (r, t, (v + 31) // 32), dtype=np.uint32)
        if t > 1:
            a["allowed"][0, 1] = 0                                      # a row without any token
    if tree:
        a["toks"] = rng.integers(0, v, (r, t)).astype(np.int32)
        a["toks"][:, ::3] = a["toks"][:, :1]
        m = rng.random((r, t, t)) < 0.4
        a["masks"] = np.stack([np.packbits(np.pad(x, ((0, 0), (0, -t % 32))), axis=1, bitorder="little").view(np.uint32) for x in m])
    return a


NAMES = dict(hist="history", hl="history_lens", pl="prompt_lens", rep="repetition", freq="frequency", pres="presence", ids="bias_ids", bias="bias",
             allowed="allowed", toks="tree_tokens", masks="tree_masks")


def call(x, a, **more):
    import torch
    from fused_turboquant_b200 import logits
    kw = {NAMES[k]: torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).cuda() for k, v in a.items() if k in NAMES}
    return logits.process(x, **kw, **more)


def lowest_best(y):
    return np.where(np.isnan(y).any(-1), np.isnan(y).argmax(-1), np.where(np.isnan(y), -np.inf, y).argmax(-1))


@pytest.mark.parametrize("r,t,v,h,k,grammar,tree", [
    (1, 1, 1, 0, 0, False, False), (1, 1, 7, 3, 2, True, False), (3, 1, 4096, 50, 0, False, False), (2, 8, 4097, 300, 5, True, True),
    (2, 3, 8192, 1, 300, True, False), (5, 4, 12344, 700, 0, False, True), (1, 33, 5000, 64, 17, True, True), (2, 256, 1000, 9, 3, False, True),
    (70, 2, 9999, 40, 1, True, False)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_process(r, t, v, h, k, grammar, tree, dtype):
    import torch
    rng = np.random.default_rng(v + r)
    a = make(rng, r, t, v, h, k, grammar, tree)
    x = torch.from_numpy(rng.normal(0, 3, (r, t, v)).astype(np.float32)).to("cuda", getattr(torch, dtype))
    x[0, 0, : v // 3] = x[0, 0, 0]                              # ties
    out, best = call(x, a)
    host = x.float().cpu().numpy()
    same, _ = plain(host, np.float32, **a)
    got = out.cpu().numpy()
    assert np.array_equal(got, same)
    assert np.array_equal(best.cpu().numpy(), lowest_best(same))
    true, size = plain(host, np.float64, **a)
    fin = np.isfinite(true)
    assert np.array_equal(fin, np.isfinite(got))
    # five roundings, each of half a unit of the largest value on the way
    assert (np.abs(got - true)[fin] <= 5 * 2.0 ** -24 * size[fin] * 1.0001).all()
    only, none = call(x, a, return_best=False)
    assert none is None and torch.equal(only, out)
    none, only = call(x, a, return_logits=False)
    assert none is None and torch.equal(only, best)


@pytest.mark.parametrize("v,stride,offset", [(1024, 1024, 0), (1024, 1032, 0), (1024, 1031, 0), (1000, 1100, 3), (1001, 1001, 0)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strides_and_alignment(v, stride, offset, dtype):
    import torch
    rng = np.random.default_rng(v + stride)
    store = torch.from_numpy(rng.normal(0, 3, 6 * stride + offset).astype(np.float32)).to("cuda", getattr(torch, dtype))
    a = make(rng, 3, 2, v, 40, 3, True, True)
    for x in (store[offset:].as_strided((3, 2, v), (2 * stride, stride, 1)), store[offset:].as_strided((3, 2, v), (stride, 3 * stride, 1)),
              store[offset:offset + 6 * v].view(3, v, 2).transpose(1, 2)):
        out, best = call(x, a)
        want, _ = plain(x.float().cpu().numpy(), np.float32, **a)
        assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(best.cpu().numpy(), lowest_best(want))


def test_two_dimensions_in_place_and_no_options():
    import torch
    from fused_turboquant_b200 import logits
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.normal(0, 3, (5, 3000)).astype(np.float32)).cuda()
    out, best = logits.process(x)
    assert torch.equal(out, x) and best.shape == (5,) and torch.equal(best.long(), x.argmax(-1))
    a = make(rng, 5, 1, 3000, 30, 4)
    want, want_best = call(x, a)
    assert want.shape == (5, 3000)
    same, same_best = call(x, a, out=x)
    assert same is x and torch.equal(x, want) and torch.equal(same_best, want_best)


def test_values_that_are_not_finite():
    import torch
    x = torch.zeros(3, 5000, device="cuda")
    x[0, 4321] = x[0, 77] = float("nan")
    x[1, 9] = float("inf")
    x[2] = -float("inf")
    hist = np.array([[77, 9, 5]] * 3, np.int32)
    a = dict(r=3, t=1, hist=hist, hl=np.full(3, 3, np.int32), rep=np.full(3, 1.5, np.float32), freq=np.ones(3, np.float32))
    out, best = call(x, a)
    want, _ = plain(x.cpu().numpy()[:, None], np.float32, **a)
    assert np.array_equal(out.cpu().numpy(), want[:, 0], equal_nan=True)
    assert best.tolist() == [77, 9, 0]
    x = torch.zeros(1, 4096 * 2, device="cuda")
    x[0, :100] = -0.0                                           # -0 and 0 are one value: the lowest index
    assert call(x, dict())[1].tolist() == [0]


@pytest.mark.parametrize("v", [9000, 9001])
def test_more_rows_of_a_request_than_a_tree_has_nodes(v):
    """600 rows without a tree: CTAs have at most 256 of them, and a warp keeps the best of 32 at a time."""
    import torch
    rng = np.random.default_rng(v)
    r, t = 2, 600
    a = make(rng, r, t, v, h=300, k=5)
    x = (8 * rng.standard_normal((r, t, v))).astype(np.float32)
    got, best = call(torch.from_numpy(x).cuda(), a)
    want, _ = plain(x, np.float32, **a)
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    np.testing.assert_array_equal(best.view(r, t).cpu().numpy(), lowest_best(want))


def test_many_repetitions_and_long_histories():
    import torch
    hist = np.full((1, 200000), 4, np.int32)
    hist[0, 1::2] = 4097
    a = dict(r=1, t=1, hist=hist, hl=np.array([200000], np.int32), pl=np.array([100], np.int32), freq=np.array([0.25], np.float32))
    out, _ = call(torch.zeros(1, 5000, device="cuda"), a)
    assert out[0, 4] == -0.25 * 99950 and out[0, 4097] == -0.25 * 99950 and float(out.abs().sum()) == 0.5 * 99950


def test_on_another_stream_and_in_a_graph():
    import torch
    rng = np.random.default_rng(5)
    a = make(rng, 4, 6, 6000, 100, 5, True, True)
    x = torch.from_numpy(rng.normal(0, 3, (4, 6, 6000)).astype(np.float32)).cuda()
    want, best = call(x, a)
    from fused_turboquant_b200 import logits
    kw = {NAMES[k]: torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).cuda() for k, v in a.items() if k in NAMES}
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, got_best = logits.process(x, **kw)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(got_best, best)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_best = logits.process(x, **kw)
    x.neg_()
    want, best = logits.process(x, **kw)
    for _ in range(3):
        graph.replay()
        assert torch.equal(got, want) and torch.equal(got_best, best)


def test_refusals():
    import torch
    from fused_turboquant_b200 import logits
    x = torch.zeros(2, 3, 64, device="cuda")
    z = lambda *s, d=torch.int32: torch.zeros(*s, dtype=d, device="cuda")  # noqa: E731
    bad = [dict(history=z(2, 4)), dict(history=z(3, 4), history_lens=z(2)), dict(history=z(2, 4), history_lens=z(3)), dict(repetition=z(3, d=torch.float32)),
           dict(bias_ids=z(2, 4)), dict(bias_ids=z(2, 4), bias=z(2, 3, d=torch.float32)), dict(allowed=z(2, 3, 1)), dict(allowed=z(2, 2, 2)),
           dict(tree_tokens=z(2, 3)), dict(tree_tokens=z(2, 3), tree_masks=z(2, 3, 2)), dict(out=z(2, 3, 63, d=torch.float32)), dict(out=z(2, 3, 64)),
           dict(return_logits=False, return_best=False)]
    for kw in bad:
        with pytest.raises(ValueError):
            logits.process(x, **kw)
    for wrong in (x[0, 0], x.double()):
        with pytest.raises(ValueError):
            logits.process(wrong)
    with pytest.raises(RuntimeError, match="CUDA"):
        logits.process(x.cpu())
    half = torch.zeros(4, 64, device="cuda", dtype=torch.float16)
    with pytest.raises(RuntimeError, match="overlaps"):
        logits.process(half, out=_alias(half))
    out, best = logits.process(torch.zeros(0, 3, 64, device="cuda"))
    assert out.shape == (0, 3, 64) and best.shape == (0, 3)


def _alias(half):
    """fp32 memory of the same shape whose first half is `half`'s."""
    import torch
    big = torch.zeros(4, 64, device="cuda")
    half.set_(big.view(-1).view(torch.float16).untyped_storage(), 0, (4, 64))
    return big


def test_graphs_with_scratch_of_their_own_run_side_by_side():
    import torch
    from fused_turboquant_b200 import logits
    r, t, v = 4, 32, 50001
    xs = [torch.randn(r, t, v, device="cuda", generator=torch.Generator("cuda").manual_seed(s)).bfloat16() for s in range(2)]
    want = [logits.process(x, return_logits=False)[1] for x in xs]
    assert logits.workspace_bytes(r * t, v) == r * t * -(-v // 2048) * 8
    assert logits.workspace_bytes(0, v) == logits.workspace_bytes(r * t, 0) == 0
    graphs, got, scratch = [], [], []
    side = torch.cuda.Stream()
    for x in xs:                                                # both captured on the same stream
        ws = torch.full((logits.workspace_bytes(r * t, v),), 255, dtype=torch.uint8, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got.append(logits.process(x, return_logits=False, workspace=ws)[1])
        graphs.append(graph)
        scratch.append(ws)
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(20):
        for best in got:
            best.fill_(-1)
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all((ws != 255).any() for ws in scratch)


def test_scratch_that_will_not_do():
    import torch
    from fused_turboquant_b200 import logits
    x = torch.randn(4, 5000, device="cuda")
    want = logits.process(x)
    need = logits.workspace_bytes(4, 5000)
    with pytest.raises(RuntimeError, match="workspace needs"):
        logits.process(x, workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="8-byte aligned"):
        logits.process(x, workspace=torch.empty(need + 8, dtype=torch.uint8, device="cuda")[4:])
    with pytest.raises(ValueError, match="workspace"):
        logits.process(x, workspace=torch.empty(need, dtype=torch.uint8))
    with pytest.raises(ValueError, match="workspace"):
        logits.process(x, workspace=torch.empty(2 * need, dtype=torch.uint8, device="cuda")[::2])
    got = logits.process(x, workspace=torch.empty(need // 8, dtype=torch.int64, device="cuda"))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    none = torch.empty(0, dtype=torch.uint8, device="cuda")     # (nothing is needed without the best tokens)
    assert torch.equal(logits.process(x, return_best=False, workspace=none)[0], want[0])
