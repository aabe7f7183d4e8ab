"""PageTable against a restatement that gives and takes pages one by one."""
import numpy as np
import pytest

from helpers import PAGE

pytestmark = pytest.mark.gpu


class Plain:
    """A page table on the host: lists, one request after the other."""

    def __init__(self, num_blocks, requests, max_blocks):
        self.rows = [[] for _ in range(requests)]
        self.lens = [0] * requests
        self.free = list(range(num_blocks - 1, -1, -1))
        self.max_blocks = max_blocks

    def extend(self, new, width, packed):
        starts, wanted, left = [0], 0, len(self.free)
        slots = np.full(width if packed else (len(new), width), -1, np.int64)
        granted = []
        for r, m in enumerate(new):
            at = starts[-1] if packed else r * width
            starts.append(at + max(m, 0) if packed else (r + 1) * width)
            n = self.lens[r]
            fits = m >= 0 and n + m <= PAGE * self.max_blocks and (at if packed else 0) + m <= width
            need = -(-(n + m) // PAGE) - -(-n // PAGE) if fits else 0
            wanted += need
            if not fits or (need and wanted > left):
                granted.append(0)
                continue
            self.rows[r] += [self.free.pop() for _ in range(need)]
            self.lens[r] = n + m
            granted.append(m)
            for j in range(m):
                slot = self.rows[r][(n + j) // PAGE] * PAGE + (n + j) % PAGE
                if packed:
                    slots[at + j] = slot
                else:
                    slots[r, j] = slot
        return slots, granted, starts

    def trim(self, keep):
        back = []
        for r, k in enumerate(keep):
            self.lens[r] = min(max(k, 0), self.lens[r])
            cut = -(-self.lens[r] // PAGE)
            back += self.rows[r][cut:]
            del self.rows[r][cut:]
        self.free += back[::-1]


def same(table, plain):
    n = int(table.n_free[0])
    assert n == len(plain.free)
    assert table.free_blocks[:n].tolist() == plain.free
    assert table.seq_lens.tolist() == plain.lens
    bt = table.block_table.cpu().numpy()
    for r, row in enumerate(plain.rows):
        assert bt[r, :len(row)].tolist() == row and (bt[r, len(row):] == -1).all()


@pytest.mark.parametrize("requests,max_blocks,num_blocks,top", [
    (1, 4, 4, 30), (3, 8, 10, 70), (33, 5, 60, 40), (700, 6, 1500, 33), (1537, 40, 20000, 300), (8192, 3, 9000, 20)])
@pytest.mark.parametrize("packed", [False, True])
def test_extend_and_trim(requests, max_blocks, num_blocks, top, packed):
    """Random steps, tables that run out of blocks, rows that are too short, numbers that are refused."""
    import torch
    from fused_turboquant_b200 import PageTable
    rng = np.random.default_rng(requests + packed)
    table, plain = PageTable(num_blocks, requests, max_blocks), Plain(num_blocks, requests, max_blocks)
    same(table, plain)
    for step in range(6):
        new = rng.integers(-1 if step else 0, top + 1, requests)
        new[rng.random(requests) < 0.2] = 0
        width = int(np.maximum(new, 0).sum() * (0.7 if step == 3 else 1) + (step == 2) * 17) if packed else int(top - (step == 3) * top // 3)
        got = table.extend(torch.tensor(new, device="cuda"), width, packed=packed)   # (int64 lengths are taken too)
        slots, granted, starts = plain.extend(new.tolist(), width, packed)
        assert got.granted.tolist() == granted and got.starts.tolist() == starts
        assert np.array_equal(got.slots.cpu().numpy(), slots)
        same(table, plain)
        keep = np.where(rng.random(requests) < 0.3, 0, np.array(plain.lens) - rng.integers(-3, 40, requests))
        table.trim(torch.tensor(keep, dtype=torch.int32, device="cuda"))
        plain.trim(keep.tolist())
        same(table, plain)


def test_giving_back_what_was_taken_restores_the_table():
    import torch
    from fused_turboquant_b200 import PageTable
    table = PageTable(500, 20, 30)
    first = torch.arange(20, dtype=torch.int32, device="cuda") * 7
    table.extend(first, 200)
    before = {k: v.clone() for k, v in table.state_dict().items()}
    table.extend(torch.full((20,), 100, dtype=torch.int32, device="cuda"), 100)
    table.trim(first)
    for k, v in table.state_dict().items():
        assert torch.equal(v, before[k]), k


def test_long_rows_and_large_slots():
    """One prompt over many CTAs' work; slots beyond 32 bits come from large block ids."""
    import torch
    from fused_turboquant_b200 import PageTable
    table = PageTable(9000, 2, 8300)
    table.free_blocks += 200_000_000
    got = table.extend(torch.tensor([131072, 9], device="cuda"), 131081, packed=True)
    want = 200_000_000 + torch.arange(131072, device="cuda") // PAGE
    assert torch.equal(got.slots[:131072], want * PAGE + torch.arange(131072, device="cuda") % PAGE)
    assert torch.equal(got.slots[131072:], (200_000_000 + 8192) * PAGE + torch.arange(9, device="cuda"))


def test_in_a_graph_and_on_another_stream():
    import torch
    from fused_turboquant_b200 import PageTable
    table, plain = PageTable(4000, 50, 80), Plain(4000, 50, 80)
    new = torch.randint(0, 20, (50,), device="cuda", dtype=torch.int32)
    back = torch.zeros(50, device="cuda", dtype=torch.int32)

    def step():
        got = table.extend(new, 20)
        table.trim(torch.maximum(table.seq_lens - back, torch.zeros_like(back)))
        return got

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    plain.extend(new.tolist(), 20, False)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    same(table, plain)
    for i in range(5):
        new.copy_(torch.randint(0, 20, (50,), device="cuda"))
        back.copy_(torch.randint(0, 30, (50,), device="cuda"))
        graph.replay()
        slots, granted, _ = plain.extend(new.tolist(), 20, False)
        plain.trim([n - b for n, b in zip(plain.lens, back.tolist())])
        assert np.array_equal(got.slots.cpu().numpy(), slots) and got.granted.tolist() == granted
        same(table, plain)


def test_refusals():
    import torch
    from fused_turboquant_b200 import PageTable
    with pytest.raises(RuntimeError, match="CUDA"):
        PageTable(4, 1, 4, device="cpu")
    with pytest.raises(ValueError, match="8192"):
        PageTable(4, 8193, 4)
    table = PageTable(4, 2, 4)
    with pytest.raises(ValueError, match="new_lens"):
        table.extend(torch.zeros(3, dtype=torch.int32, device="cuda"), 4)
    with pytest.raises(ValueError, match="width"):
        table.extend(torch.zeros(2, dtype=torch.int32, device="cuda"), -1)
    with pytest.raises(ValueError, match="keep_lens"):
        table.trim(torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="table's is"):
        table.load_state_dict(PageTable(4, 3, 4).state_dict())
    table.seq_lens = table.seq_lens.long()
    with pytest.raises(ValueError, match="int32"):
        table.trim(torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert PageTable(4, 0, 4).extend(torch.zeros(0, device="cuda"), 3).slots.shape == (0, 3)


@pytest.mark.parametrize("new,width", [
    ([2 ** 31 - 1, 2 ** 31 - 1, 5], 64), ([5, 2 ** 31 - 1, 7, 3], 64), ([2 ** 30, 2 ** 30, 2 ** 30, 2 ** 30, 3, 0], 1000),
    ([2 ** 31 - 1, 1, 1, 2 ** 31 - 2, 0, 9, -2 ** 31, 4], 40), ([3, 2 ** 31 - 1, -5, 2] + [2 ** 29] * 600 + [4, 0, 6], 30)])
def test_packed_lengths_whose_sum_passes_32_bits(new, width):
    """Requests behind the end of the slot map get nothing, however far behind it they are."""
    import torch
    from fused_turboquant_b200 import PageTable
    table, plain = PageTable(200, len(new), 4), Plain(200, len(new), 4)
    got = table.extend(torch.tensor(new, dtype=torch.int32, device="cuda"), width, packed=True)
    slots, granted, starts = plain.extend(new, width, True)
    assert got.granted.tolist() == granted and np.array_equal(got.slots.cpu().numpy(), slots)
    assert got.starts.tolist() == [min(s, 2 ** 31 - 1) for s in starts]
    same(table, plain)


@pytest.mark.parametrize("requests,width,packed", [(8192, 40, False), (8192, 200000, True), (5, 7, False)])
def test_granted_in_the_place_of_the_new_lengths(requests, width, packed):
    """C ABI: the numbers granted replace those that were asked for (many CTAs read them)."""
    import ctypes
    import torch
    from fused_turboquant_b200 import PageTable, _lib
    lib, p = _lib.load(), lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    rng = np.random.default_rng(requests)
    new = torch.tensor(rng.integers(-2, 45, requests), dtype=torch.int32, device="cuda")
    for _ in range(10):
        one, two = PageTable(12000, requests, 3), PageTable(12000, requests, 3)
        want = one.extend(new, width, packed)
        both = new.clone()
        slots = torch.zeros(want.slots.shape, dtype=torch.int64, device="cuda")
        starts = torch.zeros(requests + 1, dtype=torch.int32, device="cuda")
        rc = lib.ftq_pages_extend(p(two.block_table), p(two.seq_lens), p(two.free_blocks), p(two.n_free), requests, 3, 12000, p(both), width,
                                  int(packed), p(slots), p(both), p(starts), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0
        assert torch.equal(both, want.granted) and torch.equal(slots, want.slots) and torch.equal(starts, want.starts)
        for k, v in one.state_dict().items():
            assert torch.equal(v, two.state_dict()[k]), k


def test_numbers_of_tokens_beyond_32_bits():
    """int64 numbers: none of them wraps to a small one, or to none."""
    import torch
    from fused_turboquant_b200 import PageTable
    table = PageTable(40, 4, 8)
    big = torch.tensor([20, 2 ** 32 + 5, 2 ** 62, -2 ** 32 + 7], device="cuda")
    got = table.extend(big, 30)
    assert got.granted.tolist() == [20, 0, 0, 0] and table.seq_lens.tolist() == [20, 0, 0, 0]
    table.extend(torch.tensor([0, 9, 30, 17], device="cuda"), 30)
    before = {k: v.clone() for k, v in table.state_dict().items()}
    table.trim(torch.tensor([2 ** 32, 2 ** 62, 2 ** 31, 2 ** 63 - 1], device="cuda"))          # all that they have
    for k, v in table.state_dict().items():
        assert torch.equal(v, before[k]), k
    table.trim(torch.tensor([-2 ** 32 + 3, 4, 0, -2 ** 62], device="cuda"))
    assert table.seq_lens.tolist() == [0, 4, 0, 0] and int(table.n_free) == 39
