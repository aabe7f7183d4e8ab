"""Ancestor masks and the acceptance of drafted trees against walks on the host."""
import numpy as np
import pytest

from helpers import PAGE, page_offsets, pd

pytestmark = pytest.mark.gpu


def random_parents(rng, b, t, broken=False):
    p = np.stack([[rng.integers(0, i) if i else -1 for i in range(t)] for _ in range(b)])
    if broken:   # roots in the middle, parents that do not come first
        p[rng.random((b, t)) < 0.1] = -1
        p[rng.random((b, t)) < 0.1] = t + 3
        p[:, 0] = -7
    return p


def chain(parents, i):
    out = [i]
    while 0 <= parents[out[-1]] < out[-1]:
        out.append(int(parents[out[-1]]))
    return out


@pytest.mark.parametrize("b,t", [(1, 1), (3, 8), (5, 31), (2, 32), (4, 33), (130, 64), (2, 255), (3, 256)])
@pytest.mark.parametrize("broken", [False, True])
def test_ancestor_masks(b, t, broken):
    import torch
    from fused_turboquant_b200 import tree
    rng = np.random.default_rng(t)
    parents = random_parents(rng, b, t, broken)
    lens, ctx = rng.integers(0, t + 1, b), rng.integers(0, 1000, b)
    for tl, cl in ((None, None), (lens, ctx)):
        masks, pos = tree.ancestor_masks(torch.tensor(parents, device="cuda"), None if tl is None else torch.tensor(tl, device="cuda"),
                                         None if cl is None else torch.tensor(cl, device="cuda"))
        words = (t + 31) // 32
        want = np.zeros((b, t, words), np.uint32)
        depth = np.zeros((b, t), np.int32)
        for s in range(b):
            for i in range(t if tl is None else tl[s]):
                c = chain(parents[s], i)
                depth[s, i] = len(c) - 1
                for j in c:
                    want[s, i, j // 32] |= np.uint32(1 << (j % 32))
        assert np.array_equal(masks.cpu().numpy().view(np.uint32), want)
        assert np.array_equal(pos.cpu().numpy(), depth + (0 if cl is None else ctx[:, None]))


def test_a_chain_as_long_as_the_tree():
    import torch
    from fused_turboquant_b200 import tree
    masks, pos = tree.ancestor_masks(torch.arange(-1, 255, device="cuda")[None])
    assert pos[0].tolist() == list(range(256))
    assert masks[0, 255].tolist() == [-1] * 8 and masks[0, 31].tolist() == [-1] + [0] * 7


def walk(tokens, parents, nxt, n):
    path = [0] if n else []
    while path:
        c = path[-1]
        kids = [j for j in range(n) if parents[j] == c and parents[j] < j and tokens[j] == nxt[c]]
        if not kids:
            break
        path.append(kids[0])
    return path


def row_bytes(d, bk, bv, t):
    """Places of a token's bytes in its page, in the order of its codes."""
    kn, vc, vn, _ = page_offsets(d, bk, bv)
    k, v = np.arange(pd(d, bk)) + t * pd(d, bk), np.arange(pd(d, bv))
    if t & 2:
        v = np.roll(v, pd(d, bv) // 2)
    return np.concatenate([k, [kn + 2 * t, kn + 2 * t + 1], vc + t * pd(d, bv) + v, [vn + 2 * t, vn + 2 * t + 1]])


SHAPES = [(128, 4, 4, 8, 3, 4, 16), (64, 3, 3, 2, 2, 3, 25), (64, 2, 3, 1, 1, 5, 8), (256, 4, 2, 3, 2, 2, 33),
          (256, 4, 4, 1, 1, 2, 64), (128, 3, 4, 4, 5, 2, 200), (64, 4, 2, 2, 2, 1, 1), (128, 2, 2, 2, 40, 9, 256)]


def commit(rng, d, bk, bv, hkv, layers, ctx, lens, parents, tokens, nxt, ragged):
    """Runs the operator and the walk; how many tokens moved."""
    import torch
    from fused_turboquant_b200 import PagedKVPool
    b, t = tokens.shape
    width = (50 + t) // PAGE + 2
    nb = b * width
    table = rng.permutation(nb).reshape(b, width).astype(np.int32)
    pool = PagedKVPool(nb, hkv, d, bk, bv, n_layers=layers)
    data = rng.integers(0, 256, pool.pool.shape, dtype=np.uint8)
    pool.pool.copy_(torch.from_numpy(data))
    cu = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    seq = cu(ctx + lens)
    got = pool.tree_commit(cu(table), seq, cu(tokens), cu(parents), cu(nxt), tree_lens=cu(lens) if ragged else None)
    want = data.copy()
    moved = 0
    for s in range(b):
        path = walk(tokens[s], parents[s], nxt[s], lens[s])
        assert got.path[s].tolist() == path + [-1] * (t - len(path))
        assert got.tokens[s].tolist() == [int(nxt[s, c]) for c in path] + [-1] * (t - len(path))
        assert int(got.n_accepted[s]) == len(path) and int(got.seq_lens[s]) == ctx[s] + len(path)
        for k, c in enumerate(path):
            src, dst = ctx[s] + c, ctx[s] + k
            moved += src != dst
            want[:, table[s, dst // PAGE], :, row_bytes(d, bk, bv, dst % PAGE)] = data[:, table[s, src // PAGE], :, row_bytes(d, bk, bv, src % PAGE)]
    assert np.array_equal(pool.pool.cpu().numpy(), want)
    assert seq.tolist() == (ctx + lens).tolist()
    return moved


@pytest.mark.parametrize("d,bk,bv,hkv,layers,b,t", SHAPES)
@pytest.mark.parametrize("ragged", [False, True])
def test_tree_commit(d, bk, bv, hkv, layers, b, t, ragged):
    """Sequences without a tree or context, twins, a chain that is accepted whole, parents that are none."""
    rng = np.random.default_rng(d + t)
    lens = rng.integers(0, t + 1, b) if ragged else np.full(b, t)
    ctx = rng.integers(0, 50, b)
    ctx[0] = 0
    parents, tokens = random_parents(rng, b, t, ragged), rng.integers(0, 3, (b, t))
    nxt = rng.integers(0, 3, (b, t))
    if b > 1 and not ragged:
        parents[1] = np.arange(-1, t - 1)
        nxt[1, :-1] = tokens[1, 1:]
    commit(rng, d, bk, bv, hkv, layers, ctx, lens, parents, tokens, nxt, ragged)


@pytest.mark.parametrize("d,bk,bv,hkv,layers,b,t", [s for s in SHAPES if s[-1] > 1])
@pytest.mark.parametrize("gap", [1, 2, 9])
def test_tree_commit_moves_long_paths(d, bk, bv, hkv, layers, b, t, gap):
    """The accepted nodes are 0, gap + 1, 2 gap + 2, ...: every distance and place in a page, many batches of a warp."""
    rng = np.random.default_rng(gap)
    parents = np.zeros((b, t), np.int64)
    parents[:, 0] = -1
    path = np.arange(0, t, gap + 1)
    parents[:, path[1:]] = path[:-1]
    tokens = np.broadcast_to(np.arange(t), (b, t)).copy()
    nxt = np.full((b, t), -5)
    nxt[:, path[:-1]] = path[1:]
    moved = commit(rng, d, bk, bv, hkv, layers, rng.integers(0, 50, b), np.full(b, t), parents, tokens, nxt, False)
    assert moved == b * (len(path) - 1)


def test_commit_does_not_follow_ids_outside_the_pool():
    import torch
    from fused_turboquant_b200 import PagedKVPool
    pool = PagedKVPool(8, 1, 64, 4, 4)
    pool.pool.random_(0, 256)
    before = pool.pool.clone()
    table = torch.tensor([[3, 99, 5], [-1, 2, 1]], dtype=torch.int32, device="cuda")
    parents = torch.tensor([[-1] + [0] * 19] * 2, dtype=torch.int32, device="cuda")
    tokens = torch.arange(20, device="cuda").repeat(2, 1)
    nxt = torch.full((2, 20), 19, dtype=torch.int32, device="cuda")
    got = pool.tree_commit(table, torch.tensor([24, 24], device="cuda"), tokens, parents, nxt)
    assert got.path[:, :3].tolist() == [[0, 19, -1]] * 2      # position 23 moves to 5: neither has both pages
    assert torch.equal(pool.pool, before)


def test_tree_refusals():
    import torch
    from fused_turboquant_b200 import PagedKVPool, tree
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    with pytest.raises(RuntimeError, match="256 nodes"):
        tree.ancestor_masks(z(1, 257))
    with pytest.raises(RuntimeError, match="256 nodes"):
        tree.ancestor_masks(z(1, 0))
    with pytest.raises(ValueError, match="parents"):
        tree.ancestor_masks(z(4))
    with pytest.raises(ValueError, match="tree_lens"):
        tree.ancestor_masks(z(2, 4), z(3))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        tree.ancestor_masks(torch.zeros(1, 4, dtype=torch.int32))
    masks, pos = tree.ancestor_masks(z(0, 4))
    assert masks.shape == (0, 4, 1) and pos.shape == (0, 4)
    pool = PagedKVPool(8, 1, 64, 4, 4)
    with pytest.raises(ValueError, match="parents"):
        pool.tree_commit(z(1, 4), z(1), z(1, 4), z(1, 5), z(1, 4))
    with pytest.raises(ValueError, match="block_table"):
        pool.tree_commit(z(2, 4), z(1), z(1, 4), z(1, 4), z(1, 4))
    with pytest.raises(RuntimeError, match="256 nodes"):
        pool.tree_commit(z(1, 40), z(1), z(1, 300), z(1, 300), z(1, 300))
