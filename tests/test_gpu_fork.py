"""Rows of a page table that share blocks, against a restatement that gives and takes blocks one by one."""
import numpy as np
import pytest

from helpers import PAGE

pytestmark = pytest.mark.gpu


class Plain:
    """A page table whose rows may share blocks, on the host."""

    def __init__(self, num_blocks, requests, max_blocks):
        self.rows = [[] for _ in range(requests)]
        self.lens = [0] * requests
        self.free = list(range(num_blocks - 1, -1, -1))
        self.num_blocks, self.max_blocks = num_blocks, max_blocks

    def extend(self, new):
        got = []
        for r, m in enumerate(new):
            need = -(-(self.lens[r] + m) // PAGE) - len(self.rows[r])
            if self.lens[r] + m > PAGE * self.max_blocks or need > len(self.free):
                got.append(0)
                continue
            self.rows[r] += [self.free.pop() for _ in range(need)]
            self.lens[r] += m
            got.append(m)
        return got

    def held(self, rows):
        n = [0] * self.num_blocks
        for row in rows:
            for b in row:
                n[b] += 1
        return n

    def fork(self, parents, keep=None):
        """parents: rows of the table, -1: none.  (pairs, done)"""
        R = len(self.rows)
        lens = [min(self.lens[p], max(keep[r], 0) if keep is not None else self.lens[p]) if p >= 0 else 0 for r, p in enumerate(parents)]
        rows = [self.rows[p][:-(-n // PAGE)] if p >= 0 else [] for p, n in zip(parents, lens)]
        held = self.held(rows)
        part = [row[-1] if n % PAGE else -1 for row, n in zip(rows, lens)]
        wants = []
        for r in range(R):
            b = part[r]
            if b >= 0 and held[b] > 1 and not (held[b] == part.count(b) and part.index(b) == r):
                wants.append(r)
        gone = list(dict.fromkeys(b for row in self.rows for b in row if held[b] == 0))
        if len(wants) > len(self.free) + len(gone):
            return [], 0
        self.free += gone[::-1]
        pairs = []
        for r in wants:
            to = self.free.pop()
            pairs.append((part[r], to))
            rows[r][-1] = to
        self.rows, self.lens = rows, lens
        return pairs, 1

    def compact(self):
        used = self.num_blocks - len(self.free)
        free = set(self.free)
        holes = [b for b in range(used) if b in free]
        movers = [b for b in range(used, self.num_blocks) if b not in free]
        to = dict(zip(movers, holes))
        self.rows = [[to.get(b, b) for b in row] for row in self.rows]
        self.free = list(range(self.num_blocks - 1, used - 1, -1))
        return list(zip(movers, holes))

    def shared_lens(self, group):
        out = []
        for g in range(0, len(self.rows), group):
            live = [r for r in range(g, g + group) if self.lens[r] > 0]
            n = 0
            while live and all(n < self.lens[r] // PAGE for r in live) and len({self.rows[r][n] for r in live}) == 1:
                n += 1
            out.append(n * PAGE)
        return out


def same(table, plain):
    n = int(table.n_free[0])
    assert n == len(plain.free)
    assert table.free_blocks[:n].tolist() == plain.free
    assert table.seq_lens.tolist() == plain.lens
    bt = table.block_table.cpu().numpy()
    for r, row in enumerate(plain.rows):
        assert bt[r, :len(row)].tolist() == row and (bt[r, len(row):] == -1).all(), r
    if table.shares is not None:
        assert table.shares.tolist() == [max(x - 1, 0) for x in plain.held(plain.rows)]


def pairs_of(copies):
    c = copies.tolist()
    n = next((i for i, (a, _) in enumerate(c) if a < 0), len(c))
    assert all(a == b == -1 for a, b in c[n:])
    return [tuple(x) for x in c[:n]]


def tables(num_blocks, requests, max_blocks):
    from fused_turboquant_b200 import PageTable
    return PageTable(num_blocks, requests, max_blocks, sharing=True), Plain(num_blocks, requests, max_blocks)


def cuda(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("requests,group,max_blocks,num_blocks", [
    (1, 1, 3, 4), (4, 4, 8, 40), (6, 3, 300, 900), (33, 11, 5, 60), (33, 0, 9, 400), (512, 8, 40, 20000), (700, 0, 6, 3000), (8192, 16, 3, 30000),
    (3, 0, 1200, 4000)])
def test_fork(requests, group, max_blocks, num_blocks):
    """Random steps: rows that become others, are cut and ended, grow; tables that run out of blocks."""
    rng = np.random.default_rng(requests + group)
    table, plain = tables(num_blocks, requests, max_blocks)
    for step in range(8):
        new = rng.integers(0, PAGE * max_blocks // 3 + 2, requests) if step < 2 else rng.integers(0, 20, requests)
        width = int(new.max())
        got = table.extend(cuda(new), width)
        assert got.granted.tolist() == plain.extend(new.tolist())
        same(table, plain)
        n = group or requests
        if step % 3 == 2 or n == 1:      # few change
            parents = np.arange(requests) % n
            some = rng.random(requests) < 0.1
            parents[some] = rng.integers(-2, n + 2, int(some.sum()))
        else:
            parents = rng.integers(0, n, requests)
            parents[rng.random(requests) < 0.1] = (-1, n, -100, 2 ** 31 - 1)[step % 4]
        keep = None if step % 2 else (np.array(plain.lens) - rng.integers(-4, 30, requests)).tolist()
        first = np.arange(requests) // n * n
        absolute = np.where((parents >= 0) & (parents < n), first + parents, -1).tolist()
        f = table.fork(cuda(parents.reshape(-1, n) if group else parents), None if keep is None else cuda(keep))
        pairs, done = plain.fork(absolute, keep)
        assert int(f.done[0]) == done
        assert pairs_of(f.copies) == pairs
        same(table, plain)
        assert table.shared_lens(n).tolist() == plain.shared_lens(n)
        if step in (3, 6):
            assert pairs_of(table.compact()) == plain.compact()
            same(table, plain)


def test_too_few_blocks_change_nothing():
    table, plain = tables(6, 4, 4)
    table.extend(cuda([20, 30, 0, 0]), 30)       # four of six blocks
    plain.extend([20, 30, 0, 0])
    before = {k: v.clone() for k, v in table.state_dict().items()}
    f = table.fork(cuda([0, 0, 0, 0]))           # row 1's two come free, three are needed: four are there
    assert int(f.done[0]) == 1 and plain.fork([0, 0, 0, 0])[1] == 1
    same(table, plain)
    table.load_state_dict(before)
    table.n_free.fill_(0)                        # and now only two
    before["n_free"].zero_()
    f = table.fork(cuda([0, 0, 0, 0]))
    assert int(f.done[0]) == 0 and (f.copies == -1).all()
    for k, v in table.state_dict().items():
        assert (v == before[k]).all(), k


def test_a_whole_block_of_another_row_is_copied():
    """A row that is cut into a block that another one has whole may not write there."""
    table, plain = tables(10, 3, 4)
    table.extend(cuda([32, 0, 0]), 32)
    plain.extend([32, 0, 0])
    f = table.fork(cuda([0, 0, 0]), cuda([32, 20, 25]))
    assert pairs_of(f.copies) == plain.fork([0, 0, 0], [32, 20, 25])[0] == [(1, 2), (1, 3)]
    same(table, plain)


def test_the_lengths_themselves_as_keep_lens():
    table, plain = tables(20, 4, 4)
    table.extend(cuda([32, 5, 40, 0]), 40)
    plain.extend([32, 5, 40, 0])
    f = table.fork(cuda([2, 0, 2, 1]), keep_lens=table.seq_lens)
    assert pairs_of(f.copies) == plain.fork([2, 0, 2, 1], list(plain.lens))[0]
    same(table, plain)


@pytest.mark.parametrize("num_blocks,requests,max_blocks", [(1, 1, 1), (2, 2, 1), (7, 3, 2), (4097, 50, 90), (70000, 300, 300)])
@pytest.mark.parametrize("sharing", [False, True])
def test_compact(num_blocks, requests, max_blocks, sharing):
    import torch
    from fused_turboquant_b200 import PageTable
    rng = np.random.default_rng(num_blocks)
    table, plain = PageTable(num_blocks, requests, max_blocks, sharing=sharing), Plain(num_blocks, requests, max_blocks)
    order = rng.permutation(num_blocks)
    table.free_blocks.copy_(torch.tensor(order))
    plain.free = order.tolist()
    for step in range(3):
        new = rng.integers(0, PAGE * max_blocks // 2 + 1, requests)
        assert table.extend(cuda(new), int(new.max())).granted.tolist() == plain.extend(new.tolist())
        if sharing:
            parents = rng.integers(-1, requests, requests)
            assert pairs_of(table.fork(cuda(parents)).copies) == plain.fork(parents.tolist())[0]
        else:
            keep = np.where(rng.random(requests) < 0.5, 0, np.array(plain.lens) - 3)
            table.trim(cuda(keep))
            back = []
            for r, k in enumerate(keep):
                plain.lens[r] = max(int(k), 0)
                cut = -(-plain.lens[r] // PAGE)
                back += plain.rows[r][cut:]
                del plain.rows[r][cut:]
            plain.free += back[::-1]
        assert pairs_of(table.compact()) == plain.compact()
        same(table, plain)
    assert pairs_of(table.compact()) == []
    same(table, plain)


@pytest.mark.parametrize("layers,hkv,d,kb,vb,num_blocks,n", [
    (1, 1, 64, 2, 2, 3, 1), (3, 2, 128, 4, 4, 50, 20), (5, 8, 256, 4, 2, 40, 13), (2, 1, 64, 3, 3, 4000, 1900)])
def test_copy_pages(layers, hkv, d, kb, vb, num_blocks, n):
    import torch
    from fused_turboquant_b200 import PagedKVPool
    pool = PagedKVPool(num_blocks, hkv, d, kb, vb, n_layers=layers)
    pool.pool.copy_(torch.randint(0, 256, pool.pool.shape, dtype=torch.uint8, device="cuda"))
    ids = torch.randperm(num_blocks)[:2 * n].view(n, 2)
    if n > 2:
        ids[1], ids[2, 0] = -1, num_blocks      # passed over
        ids[0, 0] = ids[-1, 0]                  # one block to two places
    want = pool.pool.clone()
    live = ((ids >= 0) & (ids < num_blocks)).all(1)
    want[:, ids[live, 1].cuda()] = want[:, ids[live, 0].cuda()]
    pool.copy_pages(ids.cuda())
    assert torch.equal(pool.pool, want)
    pool.copy_pages(torch.empty(0, 2, dtype=torch.int32, device="cuda"))
    assert torch.equal(pool.pool, want)


def test_a_pool_of_more_than_four_gigabytes():
    """Blocks whose bytes lie beyond 32 bits."""
    import torch
    from fused_turboquant_b200 import PagedKVPool
    pool = PagedKVPool(160000, 8, 256, 4, 4, n_layers=1)         # 5.3 GB
    pool.pool[0, 5] = 7
    pool.pool[0, 159990] = 9
    pool.copy_pages(cuda([[5, 159999], [159990, 3]]))
    assert (pool.pool[0, 159999] == 7).all() and (pool.pool[0, 3] == 9).all() and (pool.pool[0, 159998] == 0).all()


def test_refusals():
    import torch
    from fused_turboquant_b200 import PageTable, PagedKVPool
    table = PageTable(8, 4, 4)
    with pytest.raises(RuntimeError, match="sharing=True"):
        table.fork(cuda([0, 1, 2, 3]))
    both = PageTable(8, 4, 4, sharing=True)
    with pytest.raises(RuntimeError, match="fork"):
        both.trim(cuda([0, 0, 0, 0]))
    with pytest.raises(ValueError, match="share"):
        table.load_state_dict(both.state_dict())
    both.load_state_dict(table.state_dict())     # (the other way round there is nothing to lose)
    for bad in (cuda([0, 1, 2]), cuda([[0, 1, 2]]), cuda([[[0, 1, 2, 3]]])):
        with pytest.raises(ValueError, match="parents"):
            both.fork(bad)
    with pytest.raises(ValueError, match="keep_lens"):
        both.fork(cuda([0, 1, 2, 3]), cuda([1]))
    with pytest.raises(RuntimeError, match="workspace needs"):
        both.fork(cuda([0, 1, 2, 3]), workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="workspace needs"):
        both.compact(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="groups of 3"):
        both.shared_lens(3)
    pool = PagedKVPool(8, 1, 64)
    with pytest.raises(ValueError, match="copies"):
        pool.copy_pages(cuda([1, 2]))


def test_captured_and_replayed():
    """A step of fork and copies in a graph, replayed on changing parents, beside eager calls that use the stream's scratch."""
    import torch
    from fused_turboquant_b200 import PagedKVPool
    table, plain = tables(200, 12, 8)
    pool = PagedKVPool(200, 2, 64, 3, 3, n_layers=2)
    pool.pool.copy_(torch.randint(0, 256, pool.pool.shape, dtype=torch.uint8, device="cuda"))
    new = [40 + r for r in range(12)]
    table.extend(cuda(new), 51)
    plain.extend(new)
    want = pool.pool.clone()
    parents = cuda([[0, 1, 2, 3]] * 3)
    ws = torch.empty(table.fork_workspace_bytes(), dtype=torch.uint8, device="cuda")
    table.fork(parents, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f = table.fork(parents, workspace=ws)
        pool.copy_pages(f.copies)
        lens = table.shared_lens(4)
    rng = np.random.default_rng(5)
    for _ in range(5):
        p = rng.integers(0, 4, (3, 4))
        parents.copy_(cuda(p))
        graph.replay()
        pairs, done = plain.fork((p + 4 * np.arange(3)[:, None]).reshape(-1).tolist())
        for a, b in pairs:
            want[:, b] = want[:, a]
        assert pairs_of(f.copies) == pairs and done == int(f.done[0])
        assert lens.tolist() == plain.shared_lens(4)
        same(table, plain)
        assert torch.equal(pool.pool, want)
        table.extend(cuda([3] * 12), 3)
        plain.extend([3] * 12)
