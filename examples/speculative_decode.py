"""Speculative decoding over the compressed paged cache: a drafted tree per request and step, all on the GPU.

    PYTHONPATH=. python examples/speculative_decode.py [--requests 8] [--new 200] [--depth 4]

A step is what a serving engine does with a tree of drafted tokens:

    table.extend             room behind every context for the tree's nodes
    tree.ancestor_masks      masks and positions from the parents
    pool.store               the nodes' keys and values, compressed        } per layer
    pool.tree_attention      every node attends context and ancestors      }
    logits.process           penalties along each node's path, best token
    pool.tree_commit         accept a path, move its keys and values behind the context
    table.trim               give the other nodes' pages back

A request that gets no pages (`granted` 0) has no tree in this step: as `tree_lens`, `granted` says so to the masks, the
attention and the commit, and the request tries again with the next step.

The model is a small random one, whose next token mostly depends on the last, and the drafts come from what followed a
token before.  Decoding is greedy, so that the answers are those of one token a step, in fewer steps, but for near ties: products of
another shape add up in another order, and a token whose logit is within rounding of the best may take its place.
"""
import argparse
import time

import torch

from fused_turboquant_b200 import PagedKVPool, PageTable, logits, tree


class Model:
    """Two layers of attention between an embedding and a head, all random but for a leaning: after a token one of 32 others
    is likely, so that answers repeat themselves and drafts can be right."""

    def __init__(self, vocab=512, d_model=256, hq=8, hkv=2, head_dim=64, n_layers=2, seed=0):
        g = torch.Generator("cuda").manual_seed(seed)
        def w(*shape):
            return (torch.randn(*shape, device="cuda", generator=g) / shape[0] ** 0.5).bfloat16()
        self.vocab, self.hq, self.hkv, self.head_dim, self.n_layers = vocab, hq, hkv, head_dim, n_layers
        self.embed = torch.randn(vocab, d_model, device="cuda", generator=g).bfloat16()
        self.qkv = [w(d_model, (hq + 2 * hkv) * head_dim) for _ in range(n_layers)]
        self.o = [0.5 * w(hq * head_dim, d_model) for _ in range(n_layers)]
        after = torch.randint(32, (vocab,), device="cuda", generator=g)
        leaning = torch.zeros(32, d_model, device="cuda").index_add_(0, after, self.embed.float()).T / d_model ** 0.5
        self.head = 4 * w(d_model, vocab)
        self.head[:, :32] += leaning.bfloat16()


class Server:
    """Requests of one model: cache, pages, histories."""

    def __init__(self, model: Model, n_requests: int, max_len: int, repetition: float = 1.1):
        self.m, self.R = model, n_requests
        blocks = -(-(max_len + tree.MAX_NODES) // 16)
        self.max_len = 16 * blocks
        self.pool = PagedKVPool(n_requests * blocks, model.hkv, model.head_dim, 4, 4, n_layers=model.n_layers)
        self.table = PageTable(n_requests * blocks, n_requests, blocks)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.history, self.history_lens = torch.zeros(n_requests, max_len + 2 * tree.MAX_NODES, **i32), torch.zeros(n_requests, **i32)
        self.prompt_lens = torch.zeros(n_requests, **i32)
        self.repetition = torch.full((n_requests,), repetition, device="cuda")

    def step(self, tokens: torch.Tensor, parents: torch.Tensor, live: torch.Tensor | None = None):
        """(logits' best token after every node, nodes of every request: all of them, or none where it is not live or no pages
        are left for it).  Keys and values of the nodes are in the cache."""
        m, (R, T) = self.m, tokens.shape
        context = self.table.seq_lens.clone()
        want = torch.full((R,), T, dtype=torch.int32, device="cuda")
        more = self.table.extend(want if live is None else want * live, width=T)
        nodes = more.granted
        masks, _ = tree.ancestor_masks(parents, nodes, context_lens=context)
        x = m.embed[tokens.long()]
        for layer in range(m.n_layers):
            q, k, v = (x @ m.qkv[layer]).view(R, T, -1, m.head_dim).split((m.hq, m.hkv, m.hkv), dim=2)
            self.pool.store(k.reshape(R * T, m.hkv, -1), v.reshape(R * T, m.hkv, -1), more.slots.view(-1), layer=layer)
            a = self.pool.tree_attention(q.contiguous(), self.table.block_table, self.table.seq_lens, self.max_len, masks, tree_lens=nodes,
                                         layer=layer)
            x = x + a.reshape(R, T, -1) @ m.o[layer]
        _, best = logits.process(x @ m.head, history=self.history, history_lens=self.history_lens, prompt_lens=self.prompt_lens,
                                 repetition=self.repetition, tree_tokens=tokens, tree_masks=masks, return_logits=False)
        return best.view(R, T), nodes

    def remember(self, tokens: torch.Tensor, count: torch.Tensor) -> None:
        """The first count[r] of each row's tokens go behind the request's history."""
        j = torch.arange(tokens.shape[1], device="cuda")
        # (the rest goes to the last column, which no history reaches)
        at = torch.where(j < count[:, None], self.history_lens[:, None] + j, self.history.shape[1] - 1)
        self.history.scatter_(1, at.long(), tokens)
        self.history_lens += count

    def prefill(self, prompts: torch.Tensor) -> torch.Tensor:
        """Prompts [R, n <= 256], as trees that are chains; the first token of each answer."""
        R, n = prompts.shape
        self.prompt_lens.fill_(n)
        self.history_lens.zero_()
        chain = torch.arange(-1, n - 1, dtype=torch.int32, device="cuda").expand(R, n).contiguous()
        # (a prompt's tokens count as prompt, not as a path: none of its nodes is in the history yet, and only the last row matters)
        self.remember(prompts, self.prompt_lens)
        lens, self.history_lens = self.history_lens, torch.zeros_like(self.history_lens)
        best, nodes = self.step(prompts, chain)
        if int(nodes.min()) < n:
            raise RuntimeError("the pool has no pages for all prompts")
        self.history_lens = lens
        return best[:, -1].contiguous()

    def draft(self, root: torch.Tensor, depth: int):
        """A chain of what followed each token last, and beside each of its nodes what followed before that."""
        R, H = self.R, self.history.shape[1]
        j = torch.arange(H - 1, device="cuda")
        valid = j + 1 < self.history_lens[:, None]
        last, before = root, root
        chain, beside = [root], []
        for _ in range(depth):
            hit = valid & (self.history[:, :-1] == last[:, None])
            at = torch.where(hit, j, -1).amax(1)
            at2 = torch.where(hit & (j < at[:, None]), j, -1).amax(1)
            follow = lambda i: self.history.gather(1, (i.clamp(min=0) + 1)[:, None])[:, 0]
            before, last = follow(at2), follow(at)
            chain.append(last)
            beside.append(before)
        tokens = torch.stack(chain + beside, 1).contiguous()
        parents = torch.tensor([-1] + list(range(depth)) + list(range(depth)), dtype=torch.int32, device="cuda").expand(R, -1).contiguous()
        return tokens, parents

    def generate(self, prompts: torch.Tensor, n_new: int, depth: int):
        """(answers [R, n_new], steps)"""
        root = self.prefill(prompts)
        R, n = prompts.shape
        steps = 0
        while int(self.history_lens.min()) < n + n_new:
            tokens, parents = self.draft(root, depth)
            # a request that has its answer, or gets no pages, has no nodes: nothing is accepted
            best, nodes = self.step(tokens, parents, self.history_lens < n + n_new)
            if int(nodes.max()) == 0:
                raise RuntimeError("the pool has no pages for any request that wants one")
            done = self.pool.tree_commit(self.table.block_table, self.table.seq_lens, tokens, parents, best, tree_lens=nodes)
            self.remember(torch.cat([root[:, None], done.tokens[:, :-1]], 1), done.n_accepted)
            self.table.trim(torch.where(self.history_lens < n + n_new, done.seq_lens, 0))     # (an answered request ends)
            fresh = done.tokens.gather(1, (done.n_accepted - 1).clamp(min=0).long()[:, None])[:, 0]
            root = torch.where(done.n_accepted > 0, fresh, root)
            steps += 1
        return self.history[:, n:n + n_new].clone(), steps


def main():
    a = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    a.add_argument("--requests", type=int, default=8)
    a.add_argument("--prompt", type=int, default=64)
    a.add_argument("--new", type=int, default=200)
    a.add_argument("--depth", type=int, default=4)
    a = a.parse_args()
    model = Model()
    prompts = torch.randint(model.vocab, (a.requests, a.prompt), dtype=torch.int32, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    answers = {}
    for depth in (0, a.depth):
        server = Server(model, a.requests, a.prompt + a.new)
        torch.cuda.synchronize()
        start = time.perf_counter()
        answers[depth], steps = server.generate(prompts, a.new, depth)
        torch.cuda.synchronize()
        print(f"trees of {1 + 2 * depth:2d} nodes: {steps} steps, {a.new / steps:.2f} tokens a step and request, {time.perf_counter() - start:.2f} s")
    same = (answers[0] == answers[a.depth]).all(1).sum()
    print(f"{int(same)} of {a.requests} answers are the same")


if __name__ == "__main__":
    main()
