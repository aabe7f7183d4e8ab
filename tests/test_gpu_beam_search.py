"""The operators of a beam search, together: a cache of shared blocks holds for every beam what a cache of its own would."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("R,K,prompt,d,bk,bv", [(1, 4, 50, 64, 4, 4), (3, 4, 37, 128, 4, 3), (5, 3, 64, 64, 2, 2), (2, 16, 5, 256, 3, 4)])
def test_a_search_with_shared_blocks_and_with_caches_of_their_own(R, K, prompt, d, bk, bv):
    """Select, fork, copy, extend, store, attend, compact, step after step; beams die and come back; every few steps each beam's
    compressed cache is that of its tokens stored alone, bit for bit, and attention over it says the same."""
    import torch
    from fused_turboquant_b200 import PagedKVPool, PageTable, beam
    g = torch.Generator("cuda").manual_seed(K)
    V, hkv, group, layers, steps, width = 40, 2, 2, 2, 45, 8
    rows = R * K
    # a token's keys and values depend on it and its position
    keys = torch.randn(layers, V, 16 * width, hkv, d, device="cuda", generator=g).bfloat16()
    values = torch.randn(layers, V, 16 * width, hkv, d, device="cuda", generator=g).bfloat16()
    pool = PagedKVPool(rows * (width + 1), hkv, d, bk, bv, n_layers=layers)
    table = PageTable(pool.num_blocks, rows, width, sharing=True)
    texts = torch.zeros(rows, 0, dtype=torch.long, device="cuda")

    def store(tokens, lens, slots):
        """tokens [n] at positions [n] of the caches."""
        for l in range(layers):
            pool.store(keys[l, tokens, lens].contiguous(), values[l, tokens, lens].contiguous(), slots, layer=l)

    first = torch.randint(V, (R, prompt), device="cuda", generator=g)
    new = torch.zeros(R, K, dtype=torch.int32, device="cuda")
    new[:, 0] = prompt
    more = table.extend(new.view(-1), prompt)
    store(first.view(-1), torch.arange(prompt, device="cuda").repeat(R), more.slots.view(R, K, prompt)[:, 0].reshape(-1))
    texts = first.repeat_interleave(K, 0)
    scores = torch.full((R, K), -torch.inf, device="cuda")
    scores[:, 0] = 0
    for step in range(steps):
        logits = 2 * torch.randn(R, K, V, device="cuda", generator=g)
        if step % 9 == 4:       # a grammar that leaves few tokens, to the first beam only
            logits[:, 1:] = -torch.inf
            logits[:, 0, 2:] = -torch.inf
        got = beam.select(logits, scores, K)
        scores = got.scores
        f = table.fork(got.parents)
        assert int(f.done[0]) == 1
        pool.copy_pages(f.copies)
        if step % 7 == 3:
            pool.copy_pages(table.compact())
        at = (got.parents.clamp(min=0) + K * torch.arange(R, device="cuda")[:, None]).view(-1)
        alive = (got.parents >= 0).view(-1)
        texts = torch.cat([texts[at], got.tokens.view(-1, 1).clamp(min=0).long()], 1)
        lens = table.seq_lens.clone()
        more = table.extend(alive.int(), 1)
        assert torch.equal(more.granted, alive.int())
        store(texts[:, -1], lens.long(), more.slots.view(-1))
        n = table.seq_lens.tolist()
        assert n == [(prompt + step + 1) * int(a) for a in alive.tolist()]
        held = table.block_table[table.block_table >= 0].unique()
        assert len(held) + int(table.n_free) == pool.num_blocks
        if step % 11 != 10 and step != steps - 1:
            continue
        # every beam alone
        alone = PagedKVPool(rows * width, hkv, d, bk, bv, n_layers=layers)
        own = torch.arange(rows * width, dtype=torch.int32, device="cuda").view(rows, width)
        for b in range(rows):
            pos = torch.arange(n[b], device="cuda")
            for l in range(layers):
                alone.store(keys[l, texts[b, :n[b]], pos].contiguous(), values[l, texts[b, :n[b]], pos].contiguous(), own[b].long()[pos // 16] * 16 + pos % 16, layer=l)
                if n[b]:
                    for x, y in zip(pool.gather_sequence(l, table.block_table[b], n[b]), alone.gather_sequence(l, own[b], n[b])):
                        assert torch.equal(x, y), (step, b)
        shared = table.shared_lens(K)
        if step < 16 and not (step % 9 == 4):
            assert (shared >= prompt // 16 * 16).all()
        q = torch.randn(rows, hkv * group, d, device="cuda", generator=g).bfloat16()
        for l in range(layers):
            out = pool.shared_attention(q, table.block_table, table.seq_lens, 16 * width, shared, layer=l)
            want = alone.shared_attention(q, own, table.seq_lens, 16 * width, torch.zeros(rows, dtype=torch.int32, device="cuda"), layer=l)
            # the same operands; the weights stand under another maximum (a rounding of 2^-11 each way), and outputs are rounded to 2^-8
            assert ((out.float() - want.float()).norm(dim=-1) <= 2.0 ** -6 * want.float().norm(dim=-1)).all()
        assert pool.decode_status() == 0
    table.fork(torch.full((rows,), -1, device="cuda"))
    assert sorted(table.free_blocks.tolist()) == list(range(pool.num_blocks)) and int(table.n_free) == pool.num_blocks
    assert (table.shares == 0).all() and (table.block_table == -1).all()


@pytest.mark.parametrize("requests,beams,prompt", [(1, 1, 3), (3, 4, 40), (2, 5, 129)])
def test_the_example_runs(requests, beams, prompt):
    import torch
    spec = importlib.util.spec_from_file_location("beam_search", os.path.join(ROOT, "examples", "beam_search.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    model = example.Model(seed=prompt)
    prompts = torch.randint(1, model.vocab, (requests, prompt), dtype=torch.int32, device="cuda", generator=torch.Generator("cuda").manual_seed(beams))
    server = example.BeamServer(model, requests, beams, prompt + 40)
    answers, score = server.generate(prompts, 40)
    assert all(0 <= len(a) <= 40 and ((a > 0) & (a < model.vocab)).all() for a in answers)
    assert torch.isfinite(score).all() and (score < 0).all()
    assert int(server.table.n_free) == server.pool.num_blocks and server.pool.decode_status() == 0


def test_a_row_without_tokens_may_be_extended_and_forked_again():
    """Rows that end and start again: numbers of samples that change, prompts admitted where others have ended."""
    import torch
    from fused_turboquant_b200 import PageTable
    rng = np.random.default_rng(1)
    table = PageTable(60, 8, 10, sharing=True)
    i32 = dict(dtype=torch.int32, device="cuda")
    for _ in range(20):
        lens = table.seq_lens
        new = torch.tensor(rng.integers(0, 30, 8), **i32)
        table.extend(torch.where(lens == 0, new, 1), 30)
        f = table.fork(torch.tensor(rng.integers(-1, 8, 8), **i32), keep_lens=torch.tensor(rng.integers(0, 60, 8), **i32))
        held = table.block_table[table.block_table >= 0]
        count = torch.bincount(held.long(), minlength=60)
        assert torch.equal((count - 1).clamp(min=0).int(), table.shares)
        free = table.free_blocks[:int(table.n_free)]
        assert len(free) + int((count > 0).sum()) == 60 and not (count[free.long()] > 0).any()
        part = (table.seq_lens % 16 != 0).nonzero()[:, 0]
        if int(f.done[0]):      # nobody else holds a block that a row will write to
            last = table.block_table[part, (table.seq_lens[part] // 16).long()]
            assert (table.shares[last.long()] == 0).all()
