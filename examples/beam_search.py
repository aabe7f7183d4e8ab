"""Beam search over the compressed paged cache: all of a step on the GPU, the beams' common blocks held and read once.

    PYTHONPATH=. python examples/beam_search.py [--requests 8] [--beams 4] [--new 60]

Row r * K + k of the page table is beam k of request r.  A step is what a serving engine does with beams:

    beam.select              the best continuations of every request's beams, and what ending would score
    table.fork               every row becomes a copy of the beam that it goes on from; whole blocks are shared
    pool.copy_pages          the partly filled last blocks that two rows would write to
    table.extend             room for the next token
    table.shared_lens        how much of the cache a request's beams have in common
    pool.store               the token's keys and values, compressed                   } per layer
    pool.shared_attention    every beam attends its cache, common blocks once           }

and now and then `table.compact` with `pool.copy_pages`, after which the blocks in use are the first ones.  The model is a small
random one.  An answer that ends is scored by its log-probability over its length; a request's best one wins.
"""
import argparse
import time

import torch

from fused_turboquant_b200 import PagedKVPool, PageTable, beam


class Model:
    """Two layers of attention between an embedding and a head, all random; token 0 ends an answer."""

    def __init__(self, vocab=512, d_model=256, hq=8, hkv=2, head_dim=64, n_layers=2, seed=0):
        g = torch.Generator("cuda").manual_seed(seed)
        def w(*shape):
            return (torch.randn(*shape, device="cuda", generator=g) / shape[0] ** 0.5).bfloat16()
        self.vocab, self.hq, self.hkv, self.head_dim, self.n_layers = vocab, hq, hkv, head_dim, n_layers
        self.embed = torch.randn(vocab, d_model, device="cuda", generator=g).bfloat16()
        self.qkv = [w(d_model, (hq + 2 * hkv) * head_dim) for _ in range(n_layers)]
        self.o = [0.5 * w(hq * head_dim, d_model) for _ in range(n_layers)]
        self.head = 4 * w(d_model, vocab)

    def heads(self, x, layer):
        """Queries, keys and values of rows [..., d_model]."""
        return (x @ self.qkv[layer]).view(*x.shape[:-1], -1, self.head_dim).split((self.hq, self.hkv, self.hkv), dim=-2)


class BeamServer:
    """Requests of one model, K beams each: cache, pages, answers."""

    def __init__(self, model: Model, n_requests: int, beams: int, max_len: int):
        self.m, self.R, self.K = model, n_requests, beams
        self.max_blocks = -(-max_len // 16)
        self.max_len, rows = 16 * self.max_blocks, n_requests * beams
        # (a prompt's blocks are there once; a block more for every row, so that a fork always finds one)
        self.pool = PagedKVPool(rows * (self.max_blocks + 1), model.hkv, model.head_dim, 4, 4, n_layers=model.n_layers)
        self.table = PageTable(self.pool.num_blocks, rows, self.max_blocks, sharing=True)
        self.ends = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.scores = torch.full((n_requests, beams), -torch.inf, device="cuda")
        self.tokens = torch.zeros(n_requests, beams, 0, dtype=torch.int32, device="cuda")
        self.best = torch.full((n_requests,), -torch.inf, device="cuda")       # of the answers that have ended
        self.answers = [None] * n_requests

    def prefill(self, prompts: torch.Tensor) -> torch.Tensor:
        """Prompts [R, n]: they go to the first beam of every request, the only one alive.  Its logits, as those of all beams."""
        m, (R, n) = self.m, prompts.shape
        new = torch.zeros(R, self.K, dtype=torch.int32, device="cuda")
        new[:, 0] = n
        more = self.table.extend(new.view(-1), width=n)
        if int(more.granted.sum()) < R * n:
            raise RuntimeError("the pool has no pages for all prompts")
        slots = more.slots.view(R, self.K, n)[:, 0].reshape(-1)
        table, lens = self.table.block_table[::self.K].contiguous(), self.table.seq_lens[::self.K].contiguous()
        x = m.embed[prompts.long()]
        for layer in range(m.n_layers):
            q, k, v = m.heads(x, layer)
            self.pool.store(k.reshape(R * n, m.hkv, -1), v.reshape(R * n, m.hkv, -1), slots, layer=layer)
            a = self.pool.continuation_attention(q.contiguous(), table, lens, self.max_len, layer=layer)
            x = x + a.reshape(R, n, -1) @ m.o[layer]
        self.scores[:, 0] = 0
        return (x[:, -1:] @ m.head).expand(R, self.K, -1)

    def choose(self, logits: torch.Tensor) -> torch.Tensor:
        """The beams' next tokens [R, K] (-1: a beam without one); rows of the page table and answers so far go with them."""
        got = beam.select(logits, self.scores, self.K, end_tokens=self.ends)
        length = self.tokens.shape[2] + 1
        # a beam that would rather end than any other continue has an answer
        ended, who = (got.end_scores[..., 0] / length).max(1)
        better = (got.end_scores.amax((1, 2)) > got.scores[:, -1]) & (ended > self.best)
        for r in better.nonzero()[:, 0].tolist():
            self.answers[r], self.best[r] = self.tokens[r, who[r]].clone(), ended[r]
        fork = self.table.fork(got.parents)
        self.pool.copy_pages(fork.copies)
        self.scores = got.scores
        from_beam = got.parents.clamp(min=0).long()[..., None].expand(-1, -1, length - 1)
        self.tokens = torch.cat([self.tokens.gather(1, from_beam), got.tokens[..., None]], -1)
        return got.tokens

    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """Logits [R, K, V] after one more token of every beam."""
        m, rows = self.m, self.R * self.K
        more = self.table.extend((tokens >= 0).int().view(-1), width=1)
        shared = self.table.shared_lens(self.K)
        x = m.embed[tokens.view(-1).clamp(min=0).long()]
        for layer in range(m.n_layers):
            q, k, v = m.heads(x, layer)
            self.pool.store(k.contiguous(), v.contiguous(), more.slots.view(-1), layer=layer)
            a = self.pool.shared_attention(q.contiguous(), self.table.block_table, self.table.seq_lens, self.max_len, shared, layer=layer)
            x = x + a.reshape(rows, -1) @ m.o[layer]
        return (x @ m.head).view(self.R, self.K, -1)

    def generate(self, prompts: torch.Tensor, n_new: int, compact_every: int = 16):
        """(answers, their log-probability over their length): ended ones, or the best beam where none has."""
        logits = self.prefill(prompts)
        for i in range(n_new):
            tokens = self.choose(logits)
            if i % compact_every == compact_every - 1:
                self.pool.copy_pages(self.table.compact())
            if i + 1 < n_new:
                logits = self.step(tokens)
        mean = self.scores[:, 0] / n_new
        for r in range(self.R):
            if self.answers[r] is None or mean[r] > self.best[r]:
                self.answers[r], self.best[r] = self.tokens[r, 0].clone(), mean[r]
        self.table.fork(torch.full((self.R * self.K,), -1, device="cuda"))     # all rows end
        return self.answers, self.best


def main():
    a = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    a.add_argument("--requests", type=int, default=8)
    a.add_argument("--beams", type=int, default=4)
    a.add_argument("--prompt", type=int, default=200)
    a.add_argument("--new", type=int, default=60)
    a = a.parse_args()
    model = Model()
    prompts = torch.randint(1, model.vocab, (a.requests, a.prompt), dtype=torch.int32, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    for beams in (1, a.beams):
        server = BeamServer(model, a.requests, beams, a.prompt + a.new)
        torch.cuda.synchronize()
        start = time.perf_counter()
        answers, score = server.generate(prompts, a.new)
        torch.cuda.synchronize()
        print(f"{beams} beams: log-probability a token {float(score.mean()):.3f}, {sum(len(x) for x in answers) / len(answers):.1f} tokens an answer, "
              f"{time.perf_counter() - start:.2f} s")


if __name__ == "__main__":
    main()
