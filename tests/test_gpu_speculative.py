"""The operators of a step with drafted trees, together: the example's answers with trees are those without."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("speculative_decode", os.path.join(ROOT, "examples", "speculative_decode.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("requests,prompt,depth", [(1, 5, 3), (3, 40, 1), (6, 129, 7)])
def test_trees_change_the_number_of_steps_and_not_the_answers(example, requests, prompt, depth):
    import torch
    model, n_new = example.Model(seed=prompt), 60
    prompts = torch.randint(model.vocab, (requests, prompt), dtype=torch.int32, device="cuda", generator=torch.Generator("cuda").manual_seed(depth))
    plain = example.Server(model, requests, prompt + n_new)
    want, plain_steps = plain.generate(prompts, n_new, 0)
    assert plain_steps == n_new
    server = example.Server(model, requests, prompt + n_new)
    got, steps = server.generate(prompts, n_new, depth)
    assert steps < plain_steps
    # Keys and values of a token are the same bits either way; scores are summed in another order, so that a near tie may fall
    # the other way and change what follows: most of the answers agree from end to end, and all of them at first.
    same = (got == want).all(1)
    assert same.float().mean() >= 0.5
    assert (got[:, :8] == want[:, :8]).all()
    # every page that the answers do not need is free, and all are when the requests end
    used = server.table.max_requests * server.table.max_blocks - int(server.table.n_free)
    assert used == int(((server.table.seq_lens + 15) // 16).sum())
    server.table.trim(torch.zeros(requests, dtype=torch.int32, device="cuda"))
    assert int(server.table.n_free) == server.table.num_blocks
    assert sorted(server.table.free_blocks.tolist()) == list(range(server.table.num_blocks))
    assert server.pool.decode_status() == 0


@pytest.mark.parametrize("requests,prompt,depth", [(2, 30, 3), (5, 17, 1), (3, 64, 7)])
def test_requests_wait_for_pages_and_lose_nothing(example, requests, prompt, depth):
    """A page a step: requests that need one in the same step wait for each other, and the answers are those with pages for all."""
    import torch
    model, n_new = example.Model(seed=7), 40
    prompts = torch.randint(model.vocab, (requests, prompt), dtype=torch.int32, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    want, steps = example.Server(model, requests, prompt + n_new).generate(prompts, n_new, depth)
    tight = example.Server(model, requests, prompt + n_new)
    table, extend = tight.table, tight.table.extend
    seen = {"refused": 0, "pages": 1}

    def a_page(new_lens, width, packed=False):
        """All but one page are somewhere else while a step asks (not for the prompts)."""
        if width >= prompt:
            return extend(new_lens, width, packed)
        free, k = int(table.n_free), seen["pages"]
        hidden = table.free_blocks[:free - k].clone()
        table.free_blocks[:k] = table.free_blocks[free - k:free].clone()
        table.n_free.fill_(k)
        got = extend(new_lens, width, packed)
        left = int(table.n_free)
        table.free_blocks[left:left + len(hidden)] = hidden
        table.n_free.fill_(left + len(hidden))
        seen["refused"] += int(((new_lens > 0) & (got.granted == 0)).sum())
        return got

    table.extend = a_page
    got, more_steps = tight.generate(prompts, n_new, depth)
    assert seen["refused"] > 0 and more_steps >= steps
    assert (got[:, :8] == want[:, :8]).all() and (got == want).all(1).float().mean() >= 0.5     # (near ties, as above)
    assert int(table.n_free) == table.num_blocks and sorted(table.free_blocks.tolist()) == list(range(table.num_blocks))
    assert tight.pool.decode_status() == 0
    seen["pages"] = 0
    with pytest.raises(RuntimeError, match="no pages"):
        tight.generate(prompts, n_new, depth)


def test_the_documented_step_with_a_refused_request():
    """extend, masks, store, attention, commit, trim as documented, where the stack has pages for one of two requests."""
    import torch
    from fused_turboquant_b200 import PagedKVPool, PageTable, tree
    hkv, hq, d, T, ctx = 2, 8, 64, 20, [45, 33]
    pool, table = PagedKVPool(16, hkv, d, 4, 4), PageTable(8, 2, 8)
    i32 = dict(dtype=torch.int32, device="cuda")
    g = torch.Generator("cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731
    first = table.extend(torch.tensor(ctx, **i32), width=max(ctx))
    assert first.granted.tolist() == ctx
    n = 2 * max(ctx)
    pool.store(rand(n, hkv, d), rand(n, hkv, d), first.slots.view(-1), layer=0)
    before = pool.pool.clone()
    held = table.block_table.clone()
    context = table.seq_lens.clone()
    more = table.extend(torch.tensor([T, T], **i32), width=T)            # the two pages that are left, and one more
    nodes = more.granted
    assert nodes.tolist() == [T, 0]
    r = 1
    parents = torch.arange(-1, T - 1, **i32).repeat(2, 1)
    masks, positions = tree.ancestor_masks(parents, nodes, context_lens=context)
    assert int(masks[r].abs().sum()) == 0
    pool.store(rand(2 * T, hkv, d), rand(2 * T, hkv, d), more.slots.view(-1), layer=0)
    out = pool.tree_attention(rand(2, T, hq, d), table.block_table, table.seq_lens, 128, masks, tree_lens=nodes, layer=0)
    assert float(out[r].abs().sum()) == 0 and torch.isfinite(out).all() and float(out[1 - r].abs().sum()) > 0
    tokens = torch.arange(T, **i32).repeat(2, 1)
    nxt = torch.roll(tokens, -1, 1).contiguous()
    nxt[:, 4] = 0                                                        # the first five nodes are accepted
    done = pool.tree_commit(table.block_table, table.seq_lens, tokens, parents, nxt, tree_lens=nodes)
    assert done.n_accepted[r] == 0 and done.n_accepted[1 - r] == 5 and done.path[r].tolist() == [-1] * T
    table.trim(done.seq_lens)
    assert table.seq_lens.tolist() == [ctx[0] + 5, ctx[1]]
    pages = held[r, :-(-ctx[r] // 16)].long()
    assert torch.equal(table.block_table[r], held[r]) and torch.equal(pool.pool[:, pages], before[:, pages])


@pytest.mark.parametrize("requests,prompt,depth", [(1, 5, 3), (3, 40, 1), (6, 129, 7)])
def test_every_token_of_an_answer_is_the_best_one(example, monkeypatch, requests, prompt, depth):
    """An answer with trees, fed to the model token by token: each of its tokens has the largest logit there, or one within rounding.

    A rounding to bf16 is off by up to 2^-9 of its size, and where sums come in another order it may fall the other way, by 2^-8.  The
    queries, values, attention and sums of two layers and the embedding's path make 8 such places; each moves a logit, a sum over
    independent coordinates, by 2^-8 of the logits' own spread at most, so that together it is sqrt(8) * 2^-8 of it in the mean and
    never four times that for two logits, sqrt(2) more.  The logits' own rounding adds 2^-8 of the largest on either side.
    """
    import torch
    model, n_new = example.Model(seed=prompt), 60
    prompts = torch.randint(model.vocab, (requests, prompt), dtype=torch.int32, device="cuda", generator=torch.Generator("cuda").manual_seed(depth))
    answer, _ = example.Server(model, requests, prompt + n_new).generate(prompts, n_new, depth)
    process, seen = example.logits.process, []

    def keeping(x, **kw):
        out, best = process(x, **dict(kw, return_logits=True))
        seen.append((out[:, -1], x[:, -1].float()))
        return out, best

    monkeypatch.setattr(example.logits, "process", keeping)
    server = example.Server(model, requests, prompt + n_new)
    root = torch.full((requests, 1), -1, dtype=torch.int32, device="cuda")
    server.prefill(prompts)
    for k in range(n_new):
        y, raw = seen[-1]
        token = answer[:, k:k + 1]
        short = y.amax(1) - y.gather(1, token.long())[:, 0]
        limit = 4 * 2 ** 0.5 * 8 ** 0.5 * 2.0 ** -8 * raw.std(1) + 2 * 2.0 ** -8 * raw.abs().amax(1)
        assert (short <= limit).all(), (k, short.tolist(), limit.tolist())
        server.step(token.contiguous(), root)
        server.remember(token, torch.ones(requests, dtype=torch.int32, device="cuda"))
