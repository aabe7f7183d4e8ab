"""Attention of rows that share their leading blocks, against its definition in 64 bits.

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


@pytest.fixture(autouse=True)
def kernels_that_read_common_blocks_once(request, monkeypatch):
    """Small calls go to the decode kernel otherwise, which has tests of its own."""
    if "as_a_user_calls_it" not in request.node.name:
        from fused_turboquant_b200 import PagedKVPool
        monkeypatch.setattr(PagedKVPool, "_takes_shared_kernel", lambda *a: True)


class Case:
    """Groups of rows: ctx[r] common tokens, lens[r][k] tokens of row k (0: none; else at least the whole blocks of ctx[r])."""

    def __init__(self, seed, d, bk, bv, hkv, g, ctx, lens, dtype="bfloat16", norm=1.0, spread=0.5, q_scale=1.0, blocks=None):
        import torch
        from fused_turboquant_b200 import PagedKVPool
        rng = np.random.default_rng(seed)
        self.d, self.bk, self.bv, self.hkv, self.g = d, bk, bv, hkv, g
        self.ctx, self.lens = np.asarray(ctx), np.asarray(lens)
        R, self.K = self.lens.shape
        flat = self.lens.reshape(-1)
        self.width = max(1, -(-int(flat.max()) // PAGE))
        table = np.full((R * self.K, self.width), -1, np.int64)
        n = 0
        for r in range(R):
            whole = int(self.ctx[r]) // PAGE
            common = np.arange(n, n + whole)
            n += whole
            for k in range(self.K):
                row, pages = table[r * self.K + k], -(-int(self.lens[r, k]) // PAGE)
                row[:min(whole, pages)] = common[:pages]
                if pages > whole:
                    row[whole:pages] = np.arange(n, n + pages - whole)
                    n += pages - whole
        self.blocks = blocks or max(n, 1)
        ids = rng.permutation(self.blocks) if blocks is None else self.blocks - 1 - np.arange(max(n, 1))
        self.table = np.where(table >= 0, ids[np.maximum(table, 0)], -1).astype(np.int32)
        self.pool = PagedKVPool(self.blocks, hkv, d, bk, bv)
        used = np.unique(self.table[self.table >= 0])
        kn, vc, vn, end = page_offsets(d, bk, bv)
        data = rng.integers(0, 256, (len(used), hkv, self.pool.page_bytes), dtype=np.uint8)
        norms = (math.sqrt(d) * np.exp(spread * rng.standard_normal((2, len(used), hkv, PAGE))) * np.broadcast_to(norm, 2)[:, None, None, None]).astype(np.float16)
        data[..., kn:vc] = norms[0].view(np.uint8)
        data[..., vn:end] = norms[1].view(np.uint8)
        self.pool.pool[0, torch.from_numpy(used.astype(np.int64)).cuda()] = torch.from_numpy(data).cuda()
        self.q = (q_scale * torch.from_numpy(rng.standard_normal((R * self.K, hkv * g, d)).astype(np.float32))).to("cuda", getattr(torch, dtype))
        self.shared = self.ctx

    def args(self):
        import torch
        i32 = dict(dtype=torch.int32, device="cuda")
        return (self.q, torch.tensor(self.table, **i32), torch.tensor(self.lens.reshape(-1), **i32), int(self.lens.max()),
                torch.tensor(np.asarray(self.shared), **i32))

    def run(self, **more):
        return self.pool.shared_attention(*self.args(), **more)

    def vectors(self, b, h, which):
        """[n, d] fp64 directions and [n] norms of the keys or values of a row and head, in the rotated space."""
        import torch
        n = int(self.lens.reshape(-1)[b])
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

    def expect(self, scale=None, rows=None):
        """(outputs, allowed distance of a row) in 64 bits."""
        import torch
        d, g = self.d, self.g
        scale = d ** -0.5 if scale is None else scale
        had = torch.ones(1, 1, dtype=torch.float64, device="cuda")
        while len(had) < d:
            had = torch.cat([torch.cat([had, had], 1), torch.cat([had, -had], 1)])
        rot = torch.from_numpy(np.asarray(self.pool.signs, np.float64)).cuda()[:, None] * had / math.sqrt(d)
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        far = torch.zeros(self.q.shape[:2], dtype=torch.float64, device="cuda")
        for b in range(len(out)) if rows is None else rows:
            if self.lens.reshape(-1)[b] == 0:
                continue
            for h in range(self.hkv):
                (k, kn), (v, vn) = self.vectors(b, h, "k"), self.vectors(b, h, "v")
                q = self.q[b, h * g:(h + 1) * g].double() @ rot
                w = torch.softmax(scale * (q @ k.T) * kn, -1)
                size = scale * ((q ** 2) @ (k ** 2).T).sqrt() * kn * math.sqrt(2) * E
                r = ((w ** 2 * (v ** 2).sum(-1) * vn ** 2) * (size ** 2 + 2 * E ** 2)).sum(-1).sqrt()
                out[b, h * g:(h + 1) * g] = (w * vn) @ v @ rot.T
                far[b, h * g:(h + 1) * g] = 4 * math.sqrt(2) * r
        return out, far


def check32(case, scale=None, rows=None, **more):
    """With an fp32 output nothing but the operands is rounded; and the 16-bit output is that, rounded."""
    import torch
    out = torch.full(case.q.shape, 7.0, device="cuda")
    assert case.run(out=out, scale=scale, **more) is out
    want, far = case.expect(scale, rows)
    keep = slice(None) if rows is None else list(rows)
    off = (out.double() - want).norm(dim=-1)[keep]
    limit = (far + 1e-5 * want.norm(dim=-1) + 1e-30)[keep]
    # (norms beyond fp16's range are infinite: what they make of a row is no number on either side)
    sure = want.isfinite().all(-1)[keep]
    bad = torch.where(sure, ~(off <= limit), out.isfinite().all(-1)[keep])
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} rows, worst {(off / limit).max():.3g} times the bound, first {bad.nonzero()[0].tolist()}"
    assert torch.equal(case.run(scale=scale, **more).nan_to_num(), out.to(case.q.dtype).nan_to_num())
    assert case.pool.decode_status() == 0
    dead = torch.from_numpy(case.lens.reshape(-1) == 0).cuda()
    assert float(out[dead].abs().sum()) == 0
    return out


def beams(ctx, own, k):
    return [[c + o] * k for c, o in zip(ctx, own)]


WIDTHS = [(bk, bv) for bk in (2, 3, 4) for bv in (2, 3, 4)]


@pytest.mark.parametrize("bk,bv", WIDTHS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_code_widths(d, bk, bv):
    check32(Case(d + 10 * bk + bv, d, bk, bv, 2, 4, [300, 5, 64], beams([300, 5, 64], [30, 3, 1], 3)))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hkv,g,k", [(1, 1, 1), (2, 4, 4), (8, 4, 8), (2, 7, 5), (1, 8, 3), (3, 5, 2), (1, 16, 4), (2, 1, 16), (1, 3, 60), (4, 2, 33), (1, 40, 1), (1, 33, 3)])
def test_heads_and_groups(d, hkv, g, k):
    """Products of one to four tiles of columns, full and padded, and more blocks of columns than one."""
    check32(Case(k + g, d, 4, 4, hkv, g, [700, 0, 129], beams([700, 0, 129], [40, 77, 100], k)))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_lengths(d, dtype):
    """Common and own tokens that begin and end at every place of a page, none of either, several thousand."""
    ctx = [0, 0, 1, 15, 16, 16, 17, 31, 32, 255, 256, 500, 512, 513, 4097, 5000]
    own = [0, 1, 0, 1, 0, 1, 15, 16, 17, 33, 0, 600, 16, 1000, 7, 0]
    check32(Case(d, d, 4, 3, 2, 2, ctx, beams(ctx, own, 4), dtype=dtype))


def test_rows_that_have_ended_and_rows_of_different_length():
    rng = np.random.default_rng(3)
    ctx = rng.integers(0, 900, 20)
    lens = ctx[:, None] + rng.integers(0, 200, (20, 5))
    lens[rng.random((20, 5)) < 0.3] = 0
    lens[7] = 0
    check32(Case(4, 128, 4, 4, 2, 4, ctx, lens))


@pytest.mark.parametrize("d", [64, 256])
def test_rows_that_end_within_the_common_tokens(d):
    """More is said to be common than the shorter rows have; beyond the longest row; numbers that are no whole blocks, or negative."""
    lens = [[500, 0, 3, 480], [16, 15, 17, 1], [100, 320, 321, 319], [40, 40, 40, 40], [64, 65, 66, 67]]
    c = Case(d, d, 4, 4, 2, 4, [480, 16, 320, 32, 64], lens)
    c.shared = [499, 100000, 335, -5, 2 ** 31 - 1]
    c.table[17:20, :4] = c.table[16, :4]
    check32(c)


def test_one_group_of_many_rows_and_many_launches():
    check32(Case(8, 64, 4, 4, 1, 1, [400], [[400 + i % 37 for i in range(1000)]]))
    rng = np.random.default_rng(9)
    ctx = rng.integers(0, 60, 700)
    check32(Case(9, 64, 4, 4, 2, 2, ctx, ctx[:, None] + rng.integers(0, 40, (700, 3))))


@pytest.mark.parametrize("norm", [2.0 ** -17, 1e-3, 300.0])
@pytest.mark.parametrize("d", [64, 128])
def test_values_of_any_size(d, norm):
    """Norms of values near both ends of fp16, alike and a factor of thousands apart (keys keep their size)."""
    for spread in (0.3, 1.2):
        check32(Case(11, d, 4, 4, 1, 4, [900, 200], beams([900, 200], [50, 50], 4), norm=(0.4 / max(spread, 0.4) ** 2, norm), spread=spread))


@pytest.mark.parametrize("q_scale,scale", [(1e-2, None), (8.0, None), (1.0, 0.5), (0.0, None)])
def test_queries_and_scales(q_scale, scale):
    check32(Case(12, 128, 4, 4, 2, 4, [600, 90], beams([600, 90], [44, 5], 4), q_scale=q_scale), scale=scale)


def test_the_decode_kernel_says_the_same():
    import torch
    c = Case(13, 128, 4, 4, 8, 4, [1000, 333], beams([1000, 333], [100, 90], 4))
    out = check32(c)
    q, table, lens, top, _ = c.args()
    other = c.pool.decode_attention(q.float(), table, lens, top, layer=0)
    _, far = c.expect()
    assert ((other - out).norm(dim=-1) <= 2 * far).all()


def test_small_batches_and_a_long_one():
    """Units cut into many pieces: one group over the whole device."""
    check32(Case(14, 128, 4, 4, 1, 4, [70000], [[70100, 70010]]))
    check32(Case(15, 128, 3, 3, 8, 8, [9000], [[9001] * 4]), rows=[0, 3])
    check32(Case(16, 256, 4, 2, 2, 2, [20000, 50], beams([20000, 50], [300, 3], 4)), rows=[0, 3, 4, 7])


def test_a_pool_of_more_than_four_gigabytes():
    """Pages whose bytes lie beyond 32 bits."""
    check32(Case(17, 256, 4, 4, 8, 2, [700], [[750, 740]], blocks=140000))        # 4.7 GB


def test_queries_anywhere():
    import torch
    c = Case(18, 128, 4, 4, 2, 4, [300], [[333, 320]])
    want = c.run()
    big = torch.zeros(2, 8, 200, dtype=c.q.dtype, device="cuda")
    big[..., 5:133] = c.q
    odd = torch.zeros(c.q.numel() + 3, dtype=c.q.dtype, device="cuda")
    odd[3:] = c.q.view(-1)
    for q in (big[..., 5:133], odd[3:].view(c.q.shape)):
        c.q = q
        assert torch.equal(c.run(), want)


@pytest.mark.parametrize("bad", [-2, 10 ** 6, 2 ** 31 - 1])
def test_block_ids_outside_the_pool(bad):
    """In common tokens all rows of the group are NaN, in a row's own that row; nothing else changes."""
    import torch
    c = Case(19, 128, 4, 4, 2, 4, [300, 200], beams([300, 200], [40, 50], 3))
    good = c.run()
    table = c.table.copy()
    c.table = table.copy()
    c.table[1, 19] = bad         # (tokens 304 on)
    out = c.run()
    assert c.pool.decode_status() & 1
    assert out[1].isnan().all() and torch.equal(out[[0, 2, 3, 4, 5]], good[[0, 2, 3, 4, 5]])
    c.table = table.copy()
    c.table[3:, 2] = bad
    out = c.run()
    assert c.pool.decode_status() & 1
    assert out[3:].isnan().all() and torch.equal(out[:3], good[:3])
    c.table = table
    assert torch.equal(c.run(), good) and c.pool.decode_status() == 0


def test_captured_and_replayed():
    import torch
    c = Case(20, 64, 4, 4, 2, 4, [500, 300], beams([500, 300], [60, 70], 4))
    q, table, lens, top, shared = c.args()
    ws = torch.empty(c.pool.shared_workspace_bytes(2, 4, 8, top), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    c.pool.shared_attention(q, table, lens, top, shared, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.pool.shared_attention(q, table, lens, top, shared, out=out, workspace=ws)
    for cut in (0, 5, 40, 300):
        c.lens = np.maximum(np.array(beams([500, 300], [60, 70], 4)) - cut, 0)
        c.ctx = c.shared = np.minimum([500, 300], c.lens[:, 0])
        lens.copy_(torch.tensor(c.lens.reshape(-1)))
        shared.copy_(torch.tensor(c.shared))
        graph.replay()
        want = c.pool.shared_attention(q, table, lens, top, shared)
        assert torch.equal(out, want)
        full, far = c.expect()
        assert ((want.double() - full).norm(dim=-1) <= far + 2.0 ** -8 * full.norm(dim=-1)).all()


def test_the_same_call_gives_the_same_bits_on_any_stream():
    import torch
    c = Case(21, 128, 4, 4, 8, 4, [900, 40, 3000], beams([900, 40, 3000], [60, 70, 9], 4))
    first = c.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = c.run()
    side.synchronize()
    assert torch.equal(first, again) and torch.equal(first, c.run())


def test_refusals():
    import torch
    c = Case(22, 64, 4, 4, 2, 4, [100, 30], beams([100, 30], [5, 6], 2))
    q, table, lens, top, shared = c.args()
    call = c.pool.shared_attention
    with pytest.raises(RuntimeError, match="CUDA"):
        call(q.cpu(), table, lens, top, shared)
    with pytest.raises(RuntimeError, match="16-bit queries"):
        call(q.float(), table, lens, top, shared)
    for bad in (q[..., :32], q[0], q.double()):
        with pytest.raises(ValueError, match="q must be"):
            call(bad, table, lens, top, shared)
    with pytest.raises(ValueError, match="block_table"):
        call(q, table[:3], lens, top, shared)
    with pytest.raises(ValueError, match="seq_lens"):
        call(q, table, lens[:3], top, shared)
    for bad in (shared[:0], shared.repeat(3), shared[None]):
        with pytest.raises(ValueError, match="shared_lens"):
            call(q, table, lens, top, bad)
    with pytest.raises(ValueError, match="max_seq_len"):
        call(q, table, lens, -1, shared)
    with pytest.raises(RuntimeError, match="too narrow"):
        call(q, table, lens, 16 * table.shape[1] + 1, shared)
    with pytest.raises(IndexError, match="layer"):
        call(q, table, lens, top, shared, layer=1)
    with pytest.raises(ValueError, match="out must be"):
        call(q, table, lens, top, shared, out=torch.empty(1, 2, 3, device="cuda"))
    with pytest.raises(RuntimeError, match="workspace needs"):
        call(q, table, lens, top, shared, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="1024 rows"):
        call(q[:1].expand(1025, -1, -1), table[:1].expand(1025, -1), lens[:1].expand(1025), top, shared[:1])
    assert call(q[:0], table[:0], lens[:0], top, shared[:0]).shape == (0, 8, 64)


@pytest.mark.parametrize("hkv,g,k,ctx,groups,both", [(8, 4, 4, 900, 1, False), (2, 7, 5, 1000, 9, False), (8, 4, 8, 4096, 12, True), (2, 16, 2, 100, 3, True),
                                                     (8, 4, 1, 3000, 40, False)])
def test_as_a_user_calls_it(hkv, g, k, ctx, groups, both):
    """Calls that go to either kernel say the same, with memory of their own too; so do refusals (above: test_refusals)."""
    import torch
    c = Case(23 + k, 128 if g != 7 else 64, 4, 4, hkv, g, [ctx] * groups, beams([ctx] * groups, range(5, 5 + groups), k))
    args = c.args()
    assert c.pool._takes_shared_kernel(*args, None, None) == both
    rows = [0, k - 1, groups * k - 1]
    check32(c, rows=rows)
    ws = torch.empty(c.pool.shared_workspace_bytes(groups, k, hkv * g, args[3]), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(c.q)
    assert torch.equal(c.run(out=out, workspace=ws), c.run())


def test_refusals_as_a_user_calls_it():
    test_refusals()


def test_queries_anywhere_as_a_user_calls_it():
    test_queries_anywhere()
