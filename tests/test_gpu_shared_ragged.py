"""Shared attention of rows of different length: what lies behind a row's end is nothing to it."""
import numpy as np
import pytest

from helpers import PAGE, page_offsets
from test_gpu_shared_attention import Case, check32

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def kernels_that_read_common_blocks_once(monkeypatch):
    from fused_turboquant_b200 import PagedKVPool
    monkeypatch.setattr(PagedKVPool, "_takes_shared_kernel", lambda *a: True)


def set_norm(case, which, row, token, value):
    """The norm of a row's token, of all KV heads, keys' or values'."""
    import torch
    kn, vc, vn, end = page_offsets(case.d, case.bk, case.bv)
    at = (kn if which == "k" else vn) + 2 * (token % PAGE)
    page = case.pool.pool[0, int(case.table[row, token // PAGE])]
    page[:, at:at + 2] = torch.tensor([value], dtype=torch.float16, device="cuda").view(torch.uint8)


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("d,g", [(64, 1), (64, 6), (128, 2), (128, 6), (256, 1), (256, 4)])        # (one tile of columns and more)
def test_norms_that_are_no_numbers_behind_a_rows_end(d, g, which, value):
    """In the page in which a row ends, of tokens that are common to longer rows, and in those behind it."""
    case = Case(d + g, d, 4, 4, 2, g, [320], [[100, 321, 251, 0, 16, 1]])
    for token, fine in ((300, [0, 2, 4, 5]), (255, [0, 2, 4, 5]), (101, [0, 4, 5]), (16, [4, 5]), (1, [5])):
        set_norm(case, which, 1, token, value)
        check32(case, rows=fine)


@pytest.mark.parametrize("d,g", [(64, 6), (128, 2)])
def test_infinite_norms_take_nothing_from_small_values(d, g):
    """Values of 2^-12 keep their bits where a longer row has an infinite one in the same page."""
    case = Case(5 + d, d, 4, 4, 2, g, [320], [[100, 321, 251]], norm=(0.4, 2.0 ** -12))
    set_norm(case, "v", 1, 101, float("inf"))
    check32(case, rows=[0])


def test_block_ids_outside_the_pool_behind_a_rows_end():
    """A bad block makes no number of the rows that have tokens in it; the others' bits stay what they were."""
    import torch
    lens = [320, 16, 17, 100, 112, 113, 250, 304]
    case = Case(31, 128, 4, 4, 2, 2, [320], [lens])
    good, table = case.run(), case.table.copy()
    assert good.isfinite().all()
    for page in range(20):
        case.table = table.copy()
        case.table[:, page] = 10 ** 6
        out = case.run()
        hit = torch.tensor([n > PAGE * page for n in lens], device="cuda")
        assert out[hit].isnan().all() and torch.equal(out[~hit], good[~hit]), page
        assert case.pool.decode_status() == 1


def test_a_group_of_many_rows_over_a_long_table():
    """The most that a group may have, under a bound of lengths far beyond what there is."""
    import torch
    case = Case(41, 128, 4, 4, 8, 1, [40], [[41 + i % 5 for i in range(1024)]])
    q, table, lens, top, shared = case.args()
    want = case.pool.shared_attention(q, table, lens, top, shared)
    wide = torch.full((1024, 1 << 14), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    for bound in (16 << 13, 16 << 14):
        got = case.pool.shared_attention(q, wide, lens, bound, shared)
        full, far = case.expect(rows=range(0, 1024, 100))
        keep = list(range(0, 1024, 100))
        assert ((got.double() - full).norm(dim=-1) <= far + 2.0 ** -8 * full.norm(dim=-1))[keep].all()
        assert (got.float() - want.float()).abs().max() <= 2.0 ** -6 * want.float().abs().max()
