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
