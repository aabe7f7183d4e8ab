"""Offsets beyond 32 bits: pages at the end of a pool of more than 4 GB, logits of more than 2^32 bytes."""
import pytest

pytestmark = pytest.mark.gpu


def test_tree_attention_and_commit_in_a_pool_of_more_than_4_gb():
    import torch
    from fused_turboquant_b200 import PagedKVPool
    hkv, group, d, t, lens = 8, 4, 128, 9, [700, 130, 9]
    b, width, far = len(lens), 44, 300_000
    g = torch.Generator("cuda").manual_seed(2)
    near = PagedKVPool(b * width, hkv, d, 4, 4)
    kv = torch.randn(2, b * width * 16, hkv, d, device="cuda", generator=g).bfloat16()
    near.store(kv[0], kv[1], torch.arange(b * width * 16, device="cuda"), layer=0)
    pool = PagedKVPool(far, hkv, d, 4, 4)
    assert pool.pool.numel() > 1 << 32
    pool.pool[0, far - b * width:] = near.pool[0]
    table = torch.arange(b * width, dtype=torch.int32, device="cuda").view(b, width)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(b, t, hkv * group, d, device="cuda", generator=g).bfloat16()
    masks = torch.tensor([[(1 << (i + 1)) - 1] for i in range(t)], dtype=torch.int32, device="cuda").expand(b, t, 1).contiguous()
    want = near.tree_attention(q, table, n, max(lens), masks)
    got = pool.tree_attention(q, table + (far - b * width), n, max(lens), masks)
    assert torch.isfinite(got).all() and torch.equal(got, want)
    # a path of nodes 0, 3 and 8: their tokens move, here as there
    tokens = torch.arange(t, dtype=torch.int32, device="cuda").expand(b, t).contiguous()
    parents = torch.tensor([-1, 0, 0, 0, 1, 1, 2, 2, 3], dtype=torch.int32, device="cuda").expand(b, t).contiguous()
    nxt = torch.tensor([3, 0, 0, 8, 0, 0, 0, 0, 0], dtype=torch.int32, device="cuda").expand(b, t).contiguous()
    before = near.pool.clone()
    one = near.tree_commit(table, n, tokens, parents, nxt)
    two = pool.tree_commit(table + (far - b * width), n, tokens, parents, nxt)
    assert one.n_accepted.tolist() == [3] * b and all(torch.equal(x, y) for x, y in zip(one, two))
    assert not torch.equal(near.pool, before) and torch.equal(pool.pool[0, far - b * width:], near.pool[0])
    assert not pool.pool[0, :far - b * width].any()


def test_slots_of_a_pool_of_more_than_4_gb():
    import torch
    from fused_turboquant_b200 import PageTable
    blocks = 1 << 28                   # slots beyond 2^32
    table = PageTable(blocks, 2, 4)
    more = table.extend(torch.tensor([20, 3], dtype=torch.int32, device="cuda"), width=20)
    # the last of the stack first: block 0 on; so give the table a stack that ends with the largest ids
    assert more.slots[0, :16].tolist() == list(range(16))
    table.trim(torch.zeros(2, dtype=torch.int32, device="cuda"))
    table.free_blocks.copy_(torch.arange(blocks, dtype=torch.int32, device="cuda"))
    more = table.extend(torch.tensor([20, 3], dtype=torch.int32, device="cuda"), width=20)
    top = (blocks - 1) * 16
    assert more.slots[0].tolist() == [top + i for i in range(16)] + [top - 16 + i for i in range(4)]
    assert more.slots[1].tolist() == [top - 32 + i for i in range(3)] + [-1] * 17


def test_logits_of_more_than_4_gb():
    import torch
    from fused_turboquant_b200 import logits
    r, t, v = 9, 16, 1 << 24
    x = torch.zeros(r, t, v, dtype=torch.bfloat16, device="cuda")
    assert x.numel() * 2 > 1 << 32
    at = torch.randint(v, (r, t), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    x.scatter_(2, at[..., None], 1.0)
    none, best = logits.process(x, return_logits=False)
    assert none is None and torch.equal(best.view(r, t).long(), at)
