"""Attention of drafted trees against its definition in 64 bits.

The kernel rounds queries, centroids and weights to fp16 and adds up in fp32.  A relative rounding error is at most 2^-11 and,
taken as independent, e = 2^-11 / sqrt(3) in the mean.  With w the softmax weights, a score is off by s = scale * |q * k| * sqrt(2) * e
(queries and centroids; |q * k|: the length of the vector of products), a weighted value by |v| * sqrt(2) * e more, so a
row by r = sqrt(sum w^2 |v|^2 (s^2 + 2 e^2)) about its mean, and as much again through the common factor 1 / sum.  A row may be
off by four times r * sqrt(2), and by the output's own rounding.
"""
import math

import numpy as np
import pytest

from helpers import PAGE, page_offsets, pd

pytestmark = pytest.mark.gpu
E = 2.0 ** -11 / math.sqrt(3)


class Case:
    """A pool of random pages, and what a call needs."""

    def __init__(self, seed, d, bk, bv, hkv, group, t, ctx, tree_lens=None, dtype="bfloat16", norm=None, q_scale=1.0):
        import torch
        from fused_turboquant_b200 import PagedKVPool
        self.rng = rng = np.random.default_rng(seed)
        self.d, self.bk, self.bv, self.hkv, self.group, self.t = d, bk, bv, hkv, group, t
        self.tree_lens = np.full(len(ctx), t) if tree_lens is None else np.asarray(tree_lens)
        self.given_lens = tree_lens is not None
        self.lens = np.asarray(ctx) + self.tree_lens
        b = len(ctx)
        self.width = max(1, -(-int(self.lens.max()) // PAGE))
        nb = b * self.width
        self.table = rng.permutation(nb).reshape(b, self.width).astype(np.int32)
        self.pool = PagedKVPool(nb, hkv, d, bk, bv)
        data = rng.integers(0, 256, self.pool.pool.shape, dtype=np.uint8)
        kn, vc, vn, end = page_offsets(d, bk, bv)
        norms = (math.sqrt(d) * np.exp(0.5 * rng.standard_normal((2, 1, nb, hkv, PAGE))) * (1.0 if norm is None else norm)).astype(np.float16)
        data[..., kn:vc] = norms[0].view(np.uint8)
        data[..., vn:end] = norms[1].view(np.uint8)
        self.pool.pool.copy_(torch.from_numpy(data))
        self.q = (q_scale * torch.from_numpy(rng.standard_normal((b, t, hkv * group, d)).astype(np.float32))).to("cuda", getattr(torch, dtype))
        m = rng.random((b, t, t)) < 0.3                       # any masks will do, rows without a node among them
        m[:, ::5] = False
        self.masks = m

    def words(self):
        import torch
        m = np.pad(self.masks, ((0, 0), (0, 0), (0, -self.t % 32)))
        return torch.from_numpy(np.packbits(m, axis=-1, bitorder="little").view(np.int32)).cuda()

    def run(self, **more):
        import torch
        return self.pool.tree_attention(self.q, torch.from_numpy(self.table).cuda(), torch.tensor(self.lens, dtype=torch.int32, device="cuda"),
                                        int(self.lens.max()), self.words(),
                                        tree_lens=torch.tensor(self.tree_lens, dtype=torch.int32, device="cuda") if self.given_lens else None, **more)

    def vectors(self, b, h, which):
        """[n, d] fp64 directions and [n] norms of the keys or values of a sequence and head, in the rotated space."""
        import torch
        n = int(self.lens[b])
        kn, vc, vn, end = page_offsets(self.d, self.bk, self.bv)
        at, norm_at, bits, lev = (0, kn, self.bk, self.pool.levels_k) if which == "k" else (vc, vn, self.bv, self.pool.levels_v)
        pages = self.pool.pool[0, torch.from_numpy(self.table[b, :-(-n // PAGE)].astype(np.int64)).cuda(), h]
        rows = pages[:, at:at + PAGE * pd(self.d, bits)].reshape(-1, pd(self.d, bits), 1)
        code = (((rows >> torch.arange(8, device="cuda", dtype=torch.uint8)) & 1).reshape(-1, self.d, bits).long() << torch.arange(bits, device="cuda")).sum(-1)
        norms = pages[:, norm_at:norm_at + 2 * PAGE].contiguous().view(torch.float16).reshape(-1, 1).double()
        x = torch.from_numpy(np.asarray(lev, np.float64)).cuda()[code]
        if which == "v":
            swapped = (torch.arange(len(x), device="cuda") & 2) != 0
            x = torch.where(swapped[:, None], x.roll(self.d // 2, 1), x)
        return x[:n], norms[:n, 0]

    def expect(self, scale=None):
        """(outputs, allowed distance of a row) in 64 bits."""
        import torch
        d, g = self.d, self.group
        scale = d ** -0.5 if scale is None else scale
        had = torch.ones(1, 1, dtype=torch.float64, device="cuda")
        while len(had) < d:
            had = torch.cat([torch.cat([had, had], 1), torch.cat([had, -had], 1)])
        rot = torch.from_numpy(np.asarray(self.pool.signs, np.float64)).cuda()[:, None] * had / math.sqrt(d)
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        far = torch.zeros(self.q.shape[:3], dtype=torch.float64, device="cuda")
        for b in range(len(self.lens)):
            n, nodes = int(self.lens[b]), min(int(self.tree_lens[b]), self.t)
            if n == 0 or nodes == 0:
                continue
            see = torch.ones(nodes, n, dtype=torch.bool, device="cuda")
            see[:, n - nodes:] = torch.from_numpy(self.masks[b, :nodes, :nodes].copy()).cuda()
            for h in range(self.hkv):
                (k, kn), (v, vn) = self.vectors(b, h, "k"), self.vectors(b, h, "v")
                q = self.q[b, :nodes, h * g:(h + 1) * g].double().transpose(0, 1) @ rot                # [g, nodes, d]
                s = torch.where(see, scale * (q @ k.T) * kn, -torch.inf)
                m = s.amax(-1, keepdim=True)
                w = torch.where(see, torch.exp(s - torch.where(m == -torch.inf, 0.0, m)), 0.0)
                total = w.sum(-1, keepdim=True)
                w = w / torch.where(total == 0, 1.0, total)
                o = torch.where(w == 0, 0.0, w * vn) @ v
                size = scale * ((q ** 2) @ (k ** 2).T).sqrt() * kn * math.sqrt(2) * E
                r = ((w ** 2 * (v ** 2).sum(-1) * vn ** 2) * (size ** 2 + 2 * E ** 2)).sum(-1).sqrt()
                out[b, :nodes, h * g:(h + 1) * g] = (o @ rot.T).transpose(0, 1)
                far[b, :nodes, h * g:(h + 1) * g] = (4 * math.sqrt(2) * r).T
        return out, far


def check32(case, scale=None, **more):
    """With an fp32 output nothing but the operands is rounded; and the 16-bit output is that, rounded."""
    import torch
    out = torch.full(case.q.shape, 7.0, device="cuda")
    assert case.run(out=out, scale=scale, **more) is out
    want, far = case.expect(scale)
    off = (out.double() - want).norm(dim=-1)
    limit = far + 1e-5 * want.norm(dim=-1) + 1e-30
    # (norms beyond fp16's range are infinite: what they make of a row is no number on either side)
    sure = want.isfinite().all(-1)
    bad = torch.where(sure, ~(off <= limit) & limit.isfinite(), out.isfinite().all(-1))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} rows, worst {(off / limit).max():.3g} times the bound, first {bad.nonzero()[0].tolist()}"
    assert torch.equal(case.run(scale=scale, **more).nan_to_num(), out.to(case.q.dtype).nan_to_num())
    assert case.pool.decode_status() == 0
    return out


WIDTHS = [(bk, bv) for bk in (2, 3, 4) for bv in (2, 3, 4)]


@pytest.mark.parametrize("bk,bv", WIDTHS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_code_widths(d, bk, bv):
    check32(Case(d + 10 * bk + bv, d, bk, bv, 2, 4, 9, [300, 5]))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hkv,group,t", [(1, 1, 1), (2, 4, 4), (8, 4, 8), (2, 7, 25), (1, 8, 16), (3, 5, 13), (1, 16, 40), (2, 1, 256), (1, 3, 200), (4, 2, 64)])
def test_heads_and_trees(d, hkv, group, t):
    """Products of 16, 32, 64 and 128 rows, full and padded, and more row tiles than one."""
    check32(Case(t + group, d, 4, 4, hkv, group, t, [700, 0, 129]))


@pytest.mark.parametrize("d,t", [(64, 32), (128, 8), (128, 16), (128, 40), (256, 12)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_context_lengths(d, t, dtype):
    """Trees that begin and end at every place of a tile and a page, contexts of none to several thousand."""
    ctx = [0, 1, 15, 16, 17, 127 - t, 128 - t, 129 - t, 120, 127, 128, 129, 255, 256, 1000, 4097]
    check32(Case(d + t, d, 4, 3, 2, 2, t, [max(0, c) for c in ctx], dtype=dtype))


def test_ragged_trees_and_empty_sequences():
    lens = [0, 1, 7, 33, 40, 12, 0, 40]
    c = Case(5, 128, 4, 4, 2, 4, 40, [0, 0, 250, 1000, 3, 128, 77, 0], tree_lens=lens)
    out = check32(c)
    for b, n in enumerate(lens):
        assert float(out[b, n:].abs().sum()) == 0


def test_rows_that_attend_nothing_are_zero():
    import torch
    c = Case(6, 64, 3, 3, 2, 7, 11, [0, 0])
    out = check32(c)
    empty = torch.from_numpy(~c.masks.any(-1)).cuda()
    assert empty.any() and float(out[empty].abs().sum()) == 0


def test_ancestor_masks_and_chains():
    """With the masks of a chain this is causal attention of the last tokens."""
    import torch
    from fused_turboquant_b200 import tree
    c = Case(7, 128, 4, 4, 8, 4, 16, [500, 900, 130])
    chain = torch.arange(-1, 15, dtype=torch.int32, device="cuda").repeat(3, 1)
    c.masks = np.broadcast_to(np.tril(np.ones((16, 16), bool)), (3, 16, 16))
    masks, _ = tree.ancestor_masks(chain)
    assert torch.equal(masks, c.words())
    out = check32(c)
    args = (torch.from_numpy(c.table).cuda(), torch.tensor(c.lens, dtype=torch.int32, device="cuda"), int(c.lens.max()))
    other = c.pool.continuation_attention(c.q, *args, layer=0)
    assert (out - other.float()).norm() < 0.01 * out.norm()


@pytest.mark.parametrize("b,hkv,top", [(1100, 1, 60), (3000, 2, 20), (1024, 1, 200)])
def test_many_sequences(b, hkv, top):
    """More sequences than one launch takes."""
    rng = np.random.default_rng(b)
    check32(Case(b, 64, 2, 2, hkv, 2, 5, rng.integers(0, top, b), tree_lens=rng.integers(0, 6, b)))


def test_one_long_context_among_short_ones():
    check32(Case(9, 128, 4, 4, 2, 4, 16, [30000, 10, 300, 0, 77]))


def test_long_context_of_few_heads():
    check32(Case(10, 128, 3, 3, 1, 8, 8, [70001]))


@pytest.mark.parametrize("norm", [1e-3, 30.0, 1000.0])
@pytest.mark.parametrize("d,t", [(128, 8), (256, 20)])
def test_norms_of_any_size(norm, d, t):
    """Norms far from 1: weights times norms neither overflow nor vanish in fp16.  (The scale keeps the scores ordinary.)"""
    check32(Case(11, d, 4, 4, 2, 2, t, [600, 100], norm=norm), scale=d ** -0.5 / norm)


@pytest.mark.parametrize("q_scale", [1e-6, 1e4, 1e9])
def test_queries_of_any_size(q_scale):
    check32(Case(12, 128, 4, 4, 2, 4, 12, [600, 3], q_scale=q_scale), scale=128 ** -0.5 / q_scale)


def test_norms_that_grow_along_the_context():
    """The scales chosen at the first tiles do not fit the later ones: values, and keys whose scores pass the reference maxima."""
    import torch
    c = Case(13, 128, 4, 4, 2, 4, 16, [2000])
    kn, vc, vn, end = page_offsets(128, 4, 4)
    for blk, page in zip(c.table[0], range(10 ** 9)):
        for at, up in ((kn, 1.02 ** (page / 4)), (vn, 1.06 ** page)):
            x = c.pool.pool[0, int(blk), :, at:at + 32].contiguous().view(torch.float16)
            c.pool.pool[0, int(blk), :, at:at + 32] = (x.float() * up * (0.05 if at == vn else 1)).to(torch.float16).view(torch.uint8)
    check32(c)


def test_what_nobody_attends_may_be_anything():
    """NaN and infinite norms of nodes that no mask has, of tokens behind the sequence, and blocks that are not its own."""
    import torch
    c = Case(14, 128, 4, 4, 2, 4, 20, [250, 300])
    c.masks = c.masks.copy()
    c.masks[:, :, [3, 7, 19]] = False
    kn, vc, vn, end = page_offsets(128, 4, 4)
    want = check32(c)
    for b in range(2):
        n = int(c.lens[b])
        for pos, bad in ((n - 17, float("nan")), (n - 13, float("inf")), (n - 1, float("nan")), (n, float("nan")), (n + 1, -float("inf"))):
            if pos // PAGE < c.width:
                blk = int(c.table[b, pos // PAGE])
                for at in (kn, vn):
                    c.pool.pool[0, blk, :, at + 2 * (pos % PAGE):at + 2 * (pos % PAGE) + 2] = torch.tensor([bad], dtype=torch.float16, device="cuda").view(torch.uint8)
    out = torch.zeros_like(want)
    c.run(out=out)
    assert torch.equal(out, want)


def test_what_is_not_a_number_reaches_the_rows_that_attend_it():
    import torch
    kn, vc, vn, end = page_offsets(128, 4, 4)
    for at in (kn, vn):
        c = Case(15, 128, 4, 4, 2, 4, 20, [250])
        node = 6
        pos = 250 + node
        c.pool.pool[0, int(c.table[0, pos // PAGE]), 1, at + 2 * (pos % PAGE):at + 2 * (pos % PAGE) + 2] = torch.tensor(
            [float("nan")], dtype=torch.float16, device="cuda").view(torch.uint8)
        out = c.run()
        sees = torch.from_numpy(c.masks[0, :, node]).cuda()
        nan = out[0].isnan().flatten(-1).any(-1)                 # [t, heads]
        assert torch.equal(nan[:, 4:], sees[:, None].expand(-1, 4)) and not nan[:, :4].any()


def test_block_ids_outside_the_pool():
    import torch
    c = Case(16, 128, 4, 4, 2, 4, 20, [250, 400, 90])
    good = c.run().clone()
    assert c.pool.decode_status() == 0
    c.table = c.table.copy()
    c.table[1, 3] = 10 ** 6
    c.table[2, (90 + 8) // PAGE] = -5                            # a page of the tree: places 6 to 19
    out = c.run()
    assert c.pool.decode_status() == 1
    assert torch.equal(out[0], good[0]) and out[1].isnan().all()
    lo = (90 + 8) // PAGE * PAGE - 90
    hit = torch.from_numpy(c.masks[2, :, max(lo, 0):lo + PAGE].any(-1)).cuda()
    if lo < 0:
        hit[:] = True
    assert torch.equal(out[2].isnan().all(-1).all(-1), hit) and torch.equal(out[2][~hit], good[2][~hit])
    c.table[1, 3], c.table[2] = 0, 0
    c.run()
    assert c.pool.decode_status() == 0


def test_layers_strides_streams_and_graphs():
    import torch
    from fused_turboquant_b200 import PagedKVPool
    c = Case(17, 128, 4, 4, 2, 4, 12, [250, 400])
    want = c.run().clone()
    three = PagedKVPool(c.pool.num_blocks, 2, 128, 4, 4, n_layers=3)
    three.pool[1] = c.pool.pool[0]
    args = (torch.from_numpy(c.table).cuda(), torch.tensor(c.lens, dtype=torch.int32, device="cuda"), int(c.lens.max()), c.words())
    assert torch.equal(three.tree_attention(c.q, *args, layer=1), want)
    wide = torch.randn(2, 12, 16, 128, device="cuda").to(c.q.dtype)
    wide[:, :, ::2] = c.q
    assert torch.equal(c.pool.tree_attention(wide[:, :, ::2], *args), want)
    table = torch.zeros(2, 2 * c.width, dtype=torch.int64, device="cuda")
    table[:, ::2] = args[0]
    assert torch.equal(c.pool.tree_attention(c.q, table[:, ::2], *args[1:]), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = c.pool.tree_attention(c.q, *args)
    s.synchronize()
    assert torch.equal(got, want)
    ws = torch.empty(c.pool.tree_workspace_bytes(2, 12, 8, int(c.lens.max())), dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.pool.tree_attention(c.q, *args, out=out, workspace=ws)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    for _ in range(20):                                          # nothing is left over from one call to the next
        assert torch.equal(c.run(), want)


def test_refusals():
    import torch
    c = Case(18, 64, 4, 4, 2, 2, 6, [20])
    bt, sl, m = torch.from_numpy(c.table).cuda(), torch.tensor(c.lens, dtype=torch.int32, device="cuda"), c.words()
    run = c.pool.tree_attention
    with pytest.raises(RuntimeError, match="16-bit"):
        run(c.q.float(), bt, sl, 26, m)
    with pytest.raises(ValueError, match="fp16 or bf16"):
        run(c.q.double(), bt, sl, 26, m)
    with pytest.raises(ValueError, match="q must be"):
        run(c.q[0], bt, sl, 26, m)
    with pytest.raises(ValueError, match="q must be"):
        run(c.q[..., :32], bt, sl, 26, m)
    with pytest.raises(ValueError, match="masks"):
        run(c.q, bt, sl, 26, m[..., :0])
    with pytest.raises(ValueError, match="seq_lens"):
        run(c.q, bt, sl.repeat(2), 26, m)
    with pytest.raises(ValueError, match="tree_lens"):
        run(c.q, bt, sl, 26, m, tree_lens=sl.repeat(2))
    with pytest.raises(ValueError, match="block_table"):
        run(c.q, bt[0], sl, 26, m)
    with pytest.raises(RuntimeError, match="too narrow"):
        run(c.q, bt, sl, 2600, m)
    with pytest.raises(RuntimeError, match="Hq"):
        run(c.q[:, :, :3], bt, sl, 26, m)
    with pytest.raises(RuntimeError, match="256 nodes"):
        run(c.q.repeat(1, 43, 1, 1)[:, :257], bt, sl, 26, torch.zeros(1, 257, 9, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="workspace"):
        run(c.q, bt, sl, 26, m, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="out"):
        run(c.q, bt, sl, 26, m, out=torch.empty(1, 6, 4, 63, device="cuda"))
    with pytest.raises(IndexError):
        run(c.q, bt, sl, 26, m, layer=1)
    with pytest.raises(RuntimeError, match="CUDA"):
        run(c.q.cpu(), bt, sl, 26, m)
    assert run(c.q[:0], bt[:0], sl[:0], 26, m[:0]).shape == (0, 6, 4, 64)


@pytest.mark.parametrize("d,t", [(64, 8), (128, 8), (128, 40), (256, 8)])
@pytest.mark.parametrize("tiles", [range(0, 13), range(2, 3), range(1, 2), range(5, 9)])
def test_whole_tiles_of_ids_outside_the_pool(d, t, tiles):
    """Shares of many tiles, of which some have no page that is there: their copies are over before they began, and no other
    sequence sees anything of it."""
    import torch
    c = Case(19, d, 4, 4, 8, 2, t, [1600] * 20 + [1000] * 8)
    good = c.run().clone()
    assert c.pool.decode_status() == 0
    c.table = c.table.copy()
    lost = [3, 4, 11, 19, 27]
    for b, bad in zip(lost, (-1, 10 ** 6, c.pool.num_blocks, -2 ** 31, 2 ** 31 - 1)):
        for tile in tiles:
            c.table[b, 8 * tile:8 * tile + 8] = bad
    if tiles[0] >= 1000 // 128:
        lost.remove(27)
    for _ in range(5):
        out = c.run()
        assert c.pool.decode_status() == 1
        for b in range(28):
            assert out[b].isnan().all() if b in lost else torch.equal(out[b], good[b])


@pytest.mark.parametrize("d,t", [(64, 8), (128, 8), (128, 40), (256, 8)])
@pytest.mark.parametrize("bad", [-1, -2, -3, -2 ** 31, 2 ** 31 - 1])
def test_every_id_outside_the_pool_is_told(d, t, bad):
    import torch
    c = Case(20, d, 4, 4, 2, 2, t, [700, 600])
    good = c.run().clone()
    c.table = c.table.copy()
    for page in (0, 21, 37):
        keep = c.table[1, page]
        c.table[1, page] = bad
        out = c.run()
        assert c.pool.decode_status() == 1
        assert out[1].isnan().all() and torch.equal(out[0], good[0])
        c.table[1, page] = keep
    assert torch.equal(c.run(), good) and c.pool.decode_status() == 0


@pytest.mark.parametrize("fill", [0.0, 1e4, 1e30, 3e38, float("inf"), float("nan")])
@pytest.mark.parametrize("d,hkv,group,t", [(64, 2, 7, 25), (128, 2, 4, 8), (128, 8, 4, 16), (128, 2, 4, 40), (256, 2, 2, 12)])
def test_queries_of_missing_nodes_may_be_anything(d, hkv, group, t, fill):
    """Their rows are zero, and the rows of the nodes that exist are what they are without them."""
    import torch
    lens = [t, 1, t // 2, 0, t - 1, 3]
    c = Case(21, d, 4, 4, hkv, group, t, [300, 700, 5, 90, 128, 0], tree_lens=lens)
    for b, n in enumerate(lens):
        c.q[b, n:] = 0
    want = check32(c)
    for b, n in enumerate(lens):
        c.q[b, n:] = fill
    out = torch.full_like(want, 7.0)
    c.run(out=out)
    assert c.pool.decode_status() == 0 and torch.equal(out, want)


def test_pages_of_a_sequence_without_nodes_are_not_looked_at():
    import torch
    c = Case(22, 128, 4, 4, 2, 4, 40, [300, 700, 90], tree_lens=[40, 0, 3])
    want = c.run().clone()
    c.table = c.table.copy()
    c.table[1] = -1
    assert torch.equal(c.run(), want) and c.pool.decode_status() == 0


@pytest.mark.parametrize("q_scale", [1e5, 1e7, 1e9, 1e15, 1e28])
@pytest.mark.parametrize("d,t", [(64, 8), (128, 8), (128, 40), (256, 12)])
def test_scores_of_any_size(d, t, q_scale):
    """Scores whose unit in the last place is above one: a row is one token's value, or some with ties, and finite."""
    import torch
    c = Case(25, d, 4, 4, 2, 4, t, [600, 3, 2000], q_scale=q_scale)
    c.masks[:, np.arange(t), np.arange(t)] = True
    out = check32(c)
    assert torch.isfinite(out).all()
    # as in fp32 with the same operands: a weight of one for the largest score, so that no row is longer than the longest value
    for b in range(3):
        for h in range(2):
            (v, vn) = c.vectors(b, h, "v")
            top = (v.norm(dim=-1) * vn).max()
            assert (out[b, :, 4 * h:4 * h + 4].double().norm(dim=-1) <= 1.01 * top).all()
            assert (out[b, :, 4 * h:4 * h + 4].norm(dim=-1) > 0).all()


@pytest.mark.parametrize("dtype,sizes", [("bfloat16", (1e3, 1e5, 1e8, 1e12, 1e20, 1e30)), ("float16", (1e2, 1e4))])
@pytest.mark.parametrize("d,hkv,group,t", [(64, 2, 2, 8), (128, 2, 4, 8), (128, 2, 4, 16), (128, 2, 4, 40), (256, 2, 2, 12), (64, 1, 16, 40)])
def test_rows_of_very_different_size(d, hkv, group, t, dtype, sizes):
    """A node or a head with large queries beside ordinary ones: every row is as precise as if it were alone."""
    import torch
    for many in (False, True):
        last = None
        for size in sizes:
            c = Case(23, d, 4, 4, hkv, group, t, [300, 1000], dtype=dtype)
            big = torch.zeros(c.q.shape[:3], dtype=torch.bool, device="cuda")
            if many:                                             # half of the heads
                big[:, :, ::2] = group > 1
            else:                                                # one node
                big[:, t // 2] = True
            c.q[big] = (c.q[big].float() * size).to(c.q.dtype)
            out = check32(c)
            assert torch.isfinite(out).all()
            if last is not None and size >= 1e8:                 # (beyond a common scale the large rows do not show in the others at all)
                assert torch.equal(out[~big], last[~big])
            last = out if size >= 1e8 else None


@pytest.mark.parametrize("tiny", [1e-3, 1e-10, 1e-30])
def test_small_rows_beside_ordinary_ones(tiny):
    c = Case(24, 128, 4, 4, 2, 4, 16, [300, 1000])
    c.q[:, ::2] = (c.q[:, ::2].float() * tiny).to(c.q.dtype)
    check32(c)


def test_scratch_in_other_memory_is_refused():
    """Host memory, and every other byte of a buffer: by the attention over a tree and by the decode attention."""
    import torch
    c = Case(26, 64, 4, 4, 2, 2, 6, [20])
    bt, sl, m = torch.from_numpy(c.table).cuda(), torch.tensor(c.lens, dtype=torch.int32, device="cuda"), c.words()
    need = max(c.pool.tree_workspace_bytes(1, 6, 4, 26), c.pool.workspace_bytes(1, 4, 26, 1))
    for ws in (torch.empty(need, dtype=torch.uint8), torch.empty(2 * need, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError, match="workspace"):
            c.pool.tree_attention(c.q, bt, sl, 26, m, workspace=ws)
        with pytest.raises(ValueError, match="workspace"):
            c.pool.decode_attention(c.q[:, 0].contiguous(), bt, sl, 26, layer=0, workspace=ws)


@pytest.mark.parametrize("offset", [1, 2, 4, 7])
def test_queries_at_any_place_of_a_larger_tensor(offset):
    import torch
    c = Case(27, 128, 4, 4, 2, 4, 9, [250, 400])
    want = c.run().clone()
    big = torch.zeros(c.q.numel() + offset, dtype=c.q.dtype, device="cuda")
    big[offset:] = c.q.reshape(-1)
    c.q = big[offset:].view(c.q.shape)
    assert c.q.is_contiguous() and c.q.data_ptr() % 16 != 0
    assert torch.equal(c.run(), want)
