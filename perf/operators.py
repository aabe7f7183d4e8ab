"""Operators of speculative serving on the compressed paged cache, measured against their plain forms.

A serving engine that drafts a tree of tokens for every request does this in a step: pages are released
and assigned, the tree's keys and values are stored, every node attends the context and its own
ancestors, the logits of every node are penalised and masked, and the accepted path moves to the front.
Four operators of that step, one kind of case each:

  pages      PageTable.trim + PageTable.extend + tree.ancestor_masks: rejected tokens give their pages back, the
             next tokens get theirs; block table, slot map, ancestor masks and positions
  attention  PagedKVPool.tree_attention over one layer of the pool
  logits     logits.process: penalties for repeated tokens (the path of a node counts), biases, grammar
             masks, and the best token
  commit     PagedKVPool.tree_commit: which nodes the target model accepts, and their compressed keys and
             values moved behind the context in every layer

`run` has each in elementary torch operations and as the framework's call.  Pools are made here, in the
framework's page layout: 16 tokens of one (block, KV head) as K codes, K norms, V codes, V norms, the halves
of a V row exchanged where bit 1 of the token's place is set.
"""
import math
from functools import lru_cache, reduce

import numpy as np
import torch

own = False

PAGE = 16
SIGN_SEED = 42
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one chat on a local machine: pages and masks of a draft of eight
        dict(name="pages_single", kind="pages", requests=1, ctx=900, tree=8, packed=False),
        # a serving batch, a draft of sixteen for every request
        dict(name="pages_serving", kind="pages", requests=256, ctx=8192, tree=16, packed=False),
        # prompts of a mixed batch admitted at once, their tokens back to back
        dict(name="pages_admit", kind="pages", requests=96, ctx=2048, tree=33, packed=True),
        # one chat: a draft of eight over a short context, every microsecond shows
        dict(name="attention_single", kind="attention", batch=1, ctx=900, ragged=False, tree=8, hq=32, hkv=8,
             d=128, kb=4, vb=4, dtype="bf16"),
        # a serving batch, sixteen nodes for every sequence
        dict(name="attention_serving", kind="attention", batch=32, ctx=8192, ragged=False, tree=16, hq=32,
             hkv=8, d=128, kb=4, vb=4, dtype="bf16"),
        # a small model's mixed batch, trees of up to 25 nodes, 3-bit codes
        dict(name="attention_small_model", kind="attention", batch=40, ctx=4096, ragged=True, tree=25, hq=14,
             hkv=2, d=64, kb=3, vb=3, dtype="fp16"),
        # heads of 256 with 2-bit values, a mixed batch
        dict(name="attention_wide_heads", kind="attention", batch=24, ctx=16384, ragged=True, tree=12, hq=16,
             hkv=8, d=256, kb=4, vb=2, dtype="bf16"),
        # long documents with a large tree, GQA group 8
        dict(name="attention_long", kind="attention", batch=2, ctx=131072, ragged=False, tree=64, hq=64, hkv=8,
             d=128, kb=3, vb=3, dtype="bf16"),
        # one chat's eight nodes: penalties only
        dict(name="logits_single", kind="logits", requests=1, tree=8, vocab=32768, history=900, biases=0,
             grammar=False, dtype="bf16"),
        # a serving batch with every option
        dict(name="logits_serving", kind="logits", requests=32, tree=16, vocab=131072, history=8192, biases=100,
             grammar=True, dtype="bf16"),
        # one chat accepts a path of its eight nodes, all layers of the model
        dict(name="commit_single", kind="commit", batch=1, ctx=900, tree=8, hkv=8, d=128, kb=4, vb=4, layers=32),
        # a serving batch accepts: thirty-two sequences, all layers, widths of codes that differ
        dict(name="commit_serving", kind="commit", batch=32, ctx=600, tree=16, hkv=8, d=128, kb=4, vb=3, layers=32),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["pages", "attention", "attention", "attention", "logits", "logits", "commit"])
    if kind == "pages":
        requests = _log_int(rng, 1, 512)
        return dict(kind=kind, requests=requests, ctx=_log_int(rng, 16, min(16384, (1 << 19) // requests)),
                    tree=_log_int(rng, 1, 128), packed=rng.random() < 0.5)
    tree = _log_int(rng, 1, 128)
    if kind == "logits":
        vocab = _log_int(rng, 1000, 160000)
        requests = _log_int(rng, 1, max(1, min(64, (1 << 26) // (vocab * tree))))
        return dict(kind=kind, requests=requests, tree=tree, vocab=vocab, history=_log_int(rng, 1, 8192),
                    biases=rng.choice([0, _log_int(rng, 1, 300)]), grammar=rng.random() < 0.5,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    d, hkv = rng.choice([64, 128, 128, 128, 256]), rng.choice([1, 2, 4, 8])
    kb, vb = rng.choice([2, 3, 4, 4]), rng.choice([2, 3, 4, 4])
    if kind == "commit":
        layers = _log_int(rng, 1, 48)
        return dict(kind=kind, batch=_log_int(rng, 1, max(1, min(64, 8192 // (layers * hkv)))), ctx=_log_int(rng, 1, 600),
                    tree=min(tree, 64), hkv=hkv, d=d, kb=kb, vb=vb, layers=layers)
    group = rng.choice([1, 2, 4, 4, 7, 8, 16])
    batch = _log_int(rng, 1, 64)
    # tokens x heads of the cache and products of a pass stay below those of the longest listed case
    top = min(131072, (1 << 21) // (batch * hkv), (1 << 30) // (batch * hkv * group * tree))
    return dict(kind=kind, batch=batch, ctx=_log_int(rng, 1, max(64, top)), ragged=rng.random() < 0.4, tree=tree,
                hq=hkv * group, hkv=hkv, d=d, kb=kb, vb=vb, dtype=rng.choice(["bf16", "bf16", "fp16"]))


# ------------------------------------------------------------------ what a case is made of
def _spread(n, top, low):
    """n lengths, log-uniform in [low, top], the first the longest: a fixed mix, the same work for every seed."""
    u = torch.rand(n, generator=torch.Generator("cpu").manual_seed(20250))
    x = torch.exp(math.log(low) + u * (math.log(top) - math.log(low))).to(torch.int64).clamp(low, top)
    x[0] = top
    return x


def _contexts(case):
    """Tokens before the tree, of every sequence."""
    n = case.get("batch") or case["requests"]
    if not (case.get("ragged") or case["kind"] == "pages"):
        return torch.full((n,), case["ctx"], dtype=torch.int64)
    return _spread(n, case["ctx"], max(1, case["ctx"] // 256))


def _tree_lens(case):
    n = case.get("batch") or case["requests"]
    if not case.get("ragged"):
        return torch.full((n,), case["tree"], dtype=torch.int64)
    return _spread(n, case["tree"], max(1, case["tree"] // 4))


def _parents(case):
    """A fixed mix of random trees: a node's parent is any node before it."""
    n, t = case.get("batch") or case["requests"], case["tree"]
    u = torch.rand(n, t, generator=torch.Generator("cpu").manual_seed(77))
    p = (u * torch.arange(t)).to(torch.int64)
    p = torch.minimum(p, (torch.arange(t) - 1).clamp(min=0))
    p[:, 0] = -1
    return p


def _reach(parents):
    """[B, T, T]: node j is node i or one of its ancestors."""
    t = parents.shape[1]
    up = (parents[:, :, None] == torch.arange(t, device=parents.device)).float()
    up = up + torch.eye(t, device=parents.device)
    return reduce(lambda a, _: ((a @ a) > 0).float(), range(max(1, (t - 1).bit_length())), up) > 0


def _to_words(bits):
    """Truth values [..., n] to int32 words, bit j % 32 of word j / 32."""
    n = bits.shape[-1]
    w = (n + 31) // 32
    x = torch.zeros(*bits.shape[:-1], 32 * w, dtype=torch.int64, device=bits.device)
    x[..., :n] = bits
    x = (x.view(*bits.shape[:-1], w, 32) << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(x >= 1 << 31, x - (1 << 32), x).to(torch.int32)


def _from_words(words, n):
    return (((words[..., None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1) != 0).flatten(-2)[..., :n]


def _accepted(case):
    """Which nodes of the fixed trees the target model accepts: the deepest node's path, or three, two or one quarter of it."""
    reach = _reach(_parents(case))
    depth = reach.sum(-1)
    t = case["tree"]
    last = (depth * (t + 1) + t - torch.arange(t)).argmax(-1)
    path = reach.gather(1, last[:, None, None].expand(-1, 1, t))[:, 0]
    keep = 4 - torch.arange(len(path)) % 4
    order = path.cumsum(-1)
    return path & (order <= keep[:, None] * depth.gather(1, last[:, None]) // 4 + 1)


def _table(lens, gen):
    """Block table of shuffled blocks, as long as the longest, and the number of blocks."""
    per = ((lens + PAGE - 1) // PAGE).cuda()
    width, nb = int(per.max()), int(per.sum())
    ids = torch.randperm(nb, device="cuda", generator=gen)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(width, device="cuda") < per[:, None]] = ids.to(torch.int32)
    return table, nb


@lru_cache(maxsize=None)
def _codebook(d, bits):
    """Lloyd-Max levels and boundaries of a coordinate of a random unit vector (pdf ~ (1 - z^2)^((d - 3) / 2))."""
    grid = np.linspace(-6 / math.sqrt(d), 6 / math.sqrt(d), 50000).clip(-1, 1)
    pdf = np.maximum(1 - grid ** 2, 0) ** ((d - 3) / 2)
    pdf /= pdf.sum()
    mass, moment = np.concatenate([[0], pdf.cumsum()]), np.concatenate([[0], (pdf * grid).cumsum()])
    edges = np.interp(np.linspace(0, 1, 2 ** bits + 1), pdf.cumsum(), grid)

    def means(e, _=None):
        at = np.searchsorted(grid, e[1:-1])
        at = np.concatenate([[0], at, [len(grid)]])
        lev = np.diff(moment[at]) / np.diff(mass[at])
        return np.concatenate([e[:1], (lev[:-1] + lev[1:]) / 2, e[-1:]])

    edges = reduce(means, range(300), edges)
    at = np.concatenate([[0], np.searchsorted(grid, edges[1:-1]), [len(grid)]])
    return (np.diff(moment[at]) / np.diff(mass[at])).astype(np.float32), edges[1:-1].astype(np.float32)


def _signs(d):
    """The rotation's signs: what the pool draws from its seed."""
    bits = torch.randint(0, 2, (d,), generator=torch.Generator("cpu").manual_seed(SIGN_SEED), dtype=torch.float32)
    return (bits * 2 - 1).cuda()


def _hadamard(d):
    i = torch.arange(d, device="cuda")
    x = i[:, None] & i[None, :]
    x = x ^ (x >> 4)
    x = x ^ (x >> 2)
    x = x ^ (x >> 1)
    return 1.0 - 2.0 * (x & 1).float()


def _pack(codes, bits):
    """Codes [..., d] to bytes: an LSB-first stream of `bits` bits each."""
    x = ((codes[..., None] >> torch.arange(bits, device=codes.device, dtype=torch.uint8)) & 1).flatten(-2)
    x = x.view(*x.shape[:-1], -1, 8) << torch.arange(8, device=codes.device, dtype=torch.uint8)
    return x.sum(-1, dtype=torch.uint8)


def _rows(shape, d, bits, gen):
    """Packed codes of random directions: one of 2^15 of them for every row."""
    edges = torch.from_numpy(_codebook(d, bits)[1]).cuda()
    x = torch.randn(1 << 15, d, device="cuda", generator=gen) / math.sqrt(d)
    lib = _pack(torch.bucketize(x, edges).to(torch.uint8), bits)
    return lib[torch.randint(0, 1 << 15, shape, device="cuda", generator=gen)]


def _pool(layers, nb, hkv, d, kb, vb, gen):
    """Pages of random vectors: directions as above, norms around sqrt(d), one in fifty three times as long."""
    shape = (layers, nb, hkv, PAGE)
    n = torch.randn(2, *shape, device="cuda", generator=gen).mul(0.3).exp() * math.sqrt(d)
    n = torch.where(torch.rand(2, *shape, device="cuda", generator=gen) < 0.02, 3 * n, n).to(torch.float16)
    n = n.view(torch.uint8)
    return torch.cat([_rows(shape, d, kb, gen).flatten(3), n[0], _rows(shape, d, vb, gen).flatten(3), n[1]], -1)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    return {"pages": _prepare_pages, "attention": _prepare_attention, "logits": _prepare_logits,
            "commit": _prepare_commit}[case["kind"]](case, gen)


def _prepare_pages(case, gen):
    """Requests that hold pages for their context and a draft; how much of it stays, and what comes next."""
    ctx, t = _contexts(case), case["tree"]
    lens = ctx + t
    table, nb = _table(lens, gen)
    spare = 64 + nb // 8
    free = torch.full((nb + spare,), -1, dtype=torch.int32, device="cuda")
    free[:spare] = nb + torch.randperm(spare, device="cuda", generator=gen).to(torch.int32)
    u = torch.rand(len(lens), device="cuda", generator=gen)
    ctx, lens = ctx.cuda(), lens.cuda()
    # a draft loses some of its nodes and gets as many again; where prompts are admitted, three of four
    # requests have ended and another prompt takes their place
    keep = ctx + 1 + (u * (t - 1)).long()
    if case["packed"]:
        keep = torch.where(u < 0.75, torch.zeros_like(keep), keep)
    s = dict(case=case, keep=keep.to(torch.int32), new=(lens - keep).to(torch.int32), parents=_parents(case).to("cuda", torch.int32),
             width=int(lens.sum()) if case["packed"] else t, top=nb + spare)
    state = dict(block_table=table, seq_lens=lens.to(torch.int32), free_blocks=free,
                 n_free=torch.tensor([spare], dtype=torch.int32, device="cuda"))
    if own:   # the handle that an engine keeps
        from fused_turboquant_b200 import PageTable
        s["pages"] = PageTable(nb + spare, len(lens), table.shape[1], device="cuda")
        s["pages"].load_state_dict(state)
    else:
        s.update(state)
    return s


def _handle(pool, case):
    from fused_turboquant_b200 import PagedKVPool
    h = PagedKVPool(pool.shape[1], case["hkv"], case["d"], case["kb"], case["vb"], n_layers=len(pool), seed=SIGN_SEED,
                    device="cuda")
    h.pool.copy_(pool)
    return h


def _prepare_attention(case, gen):
    d, t, b = case["d"], case["tree"], case["batch"]
    tree_lens = _tree_lens(case)
    lens = _contexts(case) + tree_lens
    table, nb = _table(lens, gen)
    pool = _pool(1, nb, case["hkv"], d, case["kb"], case["vb"], gen)
    masks = _reach(_parents(case)) & (torch.arange(t) < tree_lens[:, None])[:, :, None]
    s = dict(case=case, table=table, lens=lens.to("cuda", torch.int32), tree_lens=tree_lens.to("cuda", torch.int32), top=int(lens.max()),
             masks=_to_words(masks).cuda(), q=torch.randn(b, t, case["hq"], d, device="cuda", generator=gen).to(DTYPES[case["dtype"]]))
    s.update(pages=pool[0], signs=_signs(d), hadamard=_hadamard(d),
             levels_k=torch.from_numpy(_codebook(d, case["kb"])[0]).cuda(), levels_v=torch.from_numpy(_codebook(d, case["vb"])[0]).cuda())
    if own:
        s["pool"] = _handle(pool, case)
    return s


def _prepare_logits(case, gen):
    r, t, v, h = case["requests"], case["tree"], case["vocab"], case["history"]

    def tokens(*shape):   # a language's tokens: few of them make up most of a text
        u = torch.rand(*shape, device="cuda", generator=gen)
        return (u ** 4 * v).long().clamp(max=v - 1).to(torch.int32)

    def uniform(lo, hi):
        return lo + (hi - lo) * torch.rand(r, device="cuda", generator=gen)

    lens = _spread(r, h, max(1, h // 16)).to("cuda", torch.int32)
    s = dict(case=case, logits=(2.5 * torch.randn(r, t, v, device="cuda", generator=gen)).to(DTYPES[case["dtype"]]),
             history=tokens(r, h), lens=lens, prompt_lens=(lens.float() * uniform(0.2, 1.0)).to(torch.int32),
             repetition=uniform(1.0, 1.5), frequency=uniform(-0.2, 0.8), presence=uniform(0.0, 0.6),
             tokens=tokens(r, t), masks=_to_words(_reach(_parents(case))).cuda())
    if case["biases"]:
        k = min(case["biases"], v)
        first, step = torch.randint(0, v, (r, 1), device="cuda", generator=gen), max(1, v // k)
        ids = (first + step * torch.arange(k, device="cuda")) % v
        s["bias_ids"] = torch.where(torch.arange(k, device="cuda") < (k - torch.arange(r, device="cuda")[:, None] % 3), ids, -1).to(torch.int32)
        s["bias"] = 6 * torch.randn(r, k, device="cuda", generator=gen)
    if case["grammar"]:
        s["allowed"] = torch.randint(-(1 << 31), 1 << 31, (r, t, (v + 31) // 32), device="cuda", generator=gen).to(torch.int32)
        s["allowed"] &= torch.randint(-(1 << 31), 1 << 31, s["allowed"].shape, device="cuda", generator=gen).to(torch.int32)
        s["allowed"][..., ::3] = -1
    return s


def _prepare_commit(case, gen):
    t, b = case["tree"], case["batch"]
    lens = _contexts(case) + t
    table, nb = _table(lens, gen)
    pool = _pool(case["layers"], nb, case["hkv"], case["d"], case["kb"], case["vb"], gen)
    # a node's token is its index and a random part; the target model's choice is an accepted child's or nobody's
    parents, taken = _parents(case).cuda(), _accepted(case).cuda()
    tokens = torch.randint(0, 1000, (b, t), device="cuda", generator=gen) * t + torch.arange(t, device="cuda")
    child = taken[:, None, :] & (parents[:, None, :] == torch.arange(t, device="cuda")[:, None])
    nxt = torch.where(child.any(-1), (child * tokens[:, None, :]).sum(-1),
                      1000 * t + torch.randint(0, 1000, (b, t), device="cuda", generator=gen))
    s = dict(case=case, table=table, lens=lens.to("cuda", torch.int32), tokens=tokens.to(torch.int32),
             parents=parents.to(torch.int32), nxt=nxt.to(torch.int32))
    s["pool"] = _handle(pool, case) if own else pool
    return s


# ------------------------------------------------------------------ a pass
def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"pages": _plain_pages, "attention": _plain_attention, "logits": _plain_logits, "commit": _plain_commit}[kind](s)
    from fused_turboquant_b200 import logits, tree
    if kind == "pages":
        p = s["pages"]
        p.trim(s["keep"])
        ext = p.extend(s["new"], s["width"], packed=s["case"]["packed"])
        masks, positions = tree.ancestor_masks(s["parents"], context_lens=s["keep"])
        return dict(slots=ext.slots, starts=ext.starts, granted=ext.granted, masks=masks, positions=positions, **p.state_dict())
    if kind == "attention":
        return dict(out=s["pool"].tree_attention(s["q"], s["table"], s["lens"], s["top"], s["masks"], tree_lens=s["tree_lens"]))
    if kind == "logits":
        x, best = logits.process(
            s["logits"], history=s["history"], history_lens=s["lens"], prompt_lens=s["prompt_lens"], repetition=s["repetition"],
            frequency=s["frequency"], presence=s["presence"], bias_ids=s.get("bias_ids"), bias=s.get("bias"), allowed=s.get("allowed"),
            tree_tokens=s["tokens"], tree_masks=s["masks"])
        return dict(logits=x, best=best)
    got = s["pool"].tree_commit(s["table"], s["lens"], s["tokens"], s["parents"], s["nxt"])
    return dict(path=got.path, accepted=got.n_accepted, tokens=got.tokens, seq_lens=got.seq_lens, pool=s["pool"].pool)


def _plain_pages(s):
    table, lens, free, n_free = s["block_table"], s["seq_lens"], s["free_blocks"], s["n_free"]
    col = torch.arange(table.shape[1], device="cuda")
    # rejected tokens: pages behind the last token that stays go back, the first of them on top
    held, kept = (lens + PAGE - 1) // PAGE, (s["keep"] + PAGE - 1) // PAGE
    gone = (col >= kept[:, None]) & (col < held[:, None])
    ids = table[gone]
    free[n_free + len(ids) - 1 - torch.arange(len(ids), device="cuda")] = ids
    n_free += len(ids)
    table[gone] = -1
    lens.copy_(s["keep"])
    # the next tokens: pages from the top of the list, request after request, while there are enough
    new, width, packed = s["new"], s["width"], s["case"]["packed"]
    starts = torch.cat([new.new_zeros(1), new.cumsum(0, dtype=torch.int32)]) if packed else \
        torch.arange(len(new) + 1, device="cuda", dtype=torch.int32) * width
    fits = (starts[:-1] + new <= width if packed else new <= width) & (new >= 0) & (lens + new <= PAGE * table.shape[1])
    want = torch.where(fits, (lens + new + PAGE - 1) // PAGE - kept, 0)
    fits &= (want.cumsum(0) <= n_free) | (want == 0)
    more = (col >= kept[:, None]) & (col < (kept + want)[:, None]) & fits[:, None]
    n = int(more.sum())
    table[more] = free[n_free - 1 - torch.arange(n, device="cuda")]
    n_free -= n
    granted = torch.where(fits, new, 0)
    if packed:
        at = torch.arange(width, device="cuda")
        row = torch.searchsorted(starts, at, right=True) - 1
        pos, ok = lens[row.clamp(max=len(new) - 1)] + at - starts[row], row < len(new)
        row = row.clamp(max=len(new) - 1)
        ok &= fits[row]
    else:
        j = torch.arange(width, device="cuda")
        pos, ok, row = lens[:, None] + j, j < granted[:, None], torch.arange(len(new), device="cuda")[:, None]
    page = table[row, torch.where(ok, pos // PAGE, 0)].long()
    slots = torch.where(ok, page * PAGE + pos % PAGE, -1)
    lens += granted
    reach = _reach(s["parents"])
    positions = s["keep"][:, None] + reach.sum(-1, dtype=torch.int32) - 1
    return dict(slots=slots, starts=starts, granted=granted, masks=_to_words(reach), positions=positions, block_table=table,
                seq_lens=lens, free_blocks=free, n_free=n_free)


def _unpack(rows, bits):
    if bits == 4:
        return torch.stack([rows & 15, rows >> 4], -1).flatten(-2)
    if bits == 2:
        return torch.stack([rows & 3, (rows >> 2) & 3, (rows >> 4) & 3, rows >> 6], -1).flatten(-2)
    w = rows.view(*rows.shape[:-1], -1, 3).int()
    w = w[..., 0] | w[..., 1] << 8 | w[..., 2] << 16
    return ((w[..., None] >> torch.arange(0, 24, 3, device=w.device)) & 7).flatten(-2)


def _plain_attention(s):
    case = s["case"]
    b, t, hq, d = s["q"].shape
    h, pdk, pdv = case["hkv"], d * case["kb"] // 8, d * case["vb"] // 8
    pages = s["pages"][s["table"].clamp(min=0).long()].transpose(1, 2)               # [B, H, blocks, bytes]
    k, kn, v, vn = pages.split([PAGE * pdk, 2 * PAGE, PAGE * pdv, 2 * PAGE], -1)

    def dense(rows, norms, levels, bits, width):
        rows = rows.reshape(b, h, -1, PAGE, width)
        x = levels[_unpack(rows, bits).int()]
        if width == pdv and bits == case["vb"] and levels is s["levels_v"]:
            odd = (torch.arange(PAGE, device="cuda") & 2 != 0)[:, None]
            x = torch.where(odd, torch.cat([x[..., d // 2:], x[..., :d // 2]], -1), x)
        return (x * norms.contiguous().view(torch.float16).float()[..., None]).flatten(2, 3)   # [B, H, S, D]

    q = (s["q"].float() * s["signs"]) @ s["hadamard"] / math.sqrt(d)
    q = q.view(b, t, h, hq // h, d).transpose(1, 2).flatten(2, 3)                     # [B, H, T * G, D]
    scores = q @ dense(k, kn, s["levels_k"], case["kb"], pdk).transpose(-1, -2) * d ** -0.5
    n = scores.shape[-1]
    pos = torch.arange(n, device="cuda")
    node = pos - (s["lens"] - s["tree_lens"])[:, None]                               # [B, S]
    bits = _from_words(s["masks"], t)                                                # [B, T, T]
    sees = bits.gather(2, node.clamp(0, t - 1)[:, None, :].expand(-1, t, -1)) | (node < 0)[:, None, :]
    sees &= (pos < s["lens"][:, None])[:, None, :] & (torch.arange(t, device="cuda") < s["tree_lens"][:, None])[:, :, None]
    sees = sees.repeat_interleave(hq // h, 1)[:, None]                                # [B, 1, T * G, S]
    scores = torch.where(sees, scores, -torch.inf)
    m = scores.amax(-1, keepdim=True)
    w = torch.where(sees, torch.exp(scores - torch.where(m == -torch.inf, 0.0, m)), 0.0)
    del scores
    total = w.sum(-1, keepdim=True)
    out = w @ dense(v, vn, s["levels_v"], case["vb"], pdv) / torch.where(total == 0, 1.0, total)
    out = (out @ s["hadamard"] / math.sqrt(d)) * s["signs"]
    return dict(out=out.view(b, h, t, hq // h, d).transpose(1, 2).reshape(b, t, hq, d).to(s["q"].dtype))


def _plain_logits(s):
    x = s["logits"].float()
    r, t, v = x.shape
    at = torch.arange(s["history"].shape[1], device="cuda")
    ids = s["history"].long()
    seen = torch.zeros(r, v, device="cuda").scatter_add_(1, ids, (at < s["prompt_lens"][:, None]).float())
    said = torch.zeros(r, v, device="cuda").scatter_add_(1, ids, ((at >= s["prompt_lens"][:, None]) & (at < s["lens"][:, None])).float())
    said = said[:, None].repeat(1, t, 1)
    said.scatter_add_(2, s["tokens"].long()[:, None].expand(-1, t, -1), _from_words(s["masks"], t).float())
    p = s["repetition"][:, None, None]
    x = torch.where((seen[:, None] > 0) | (said > 0), torch.where(x > 0, x / p, x * p), x)
    x = x - s["frequency"][:, None, None] * said
    x = x - torch.where(said > 0, s["presence"][:, None, None], 0.0)
    if "bias" in s:
        ids = s["bias_ids"].long()
        dense = torch.zeros(r, v, device="cuda").scatter_add_(1, ids.clamp(min=0), torch.where(ids >= 0, s["bias"], 0.0))
        x = x + dense[:, None]
    if "allowed" in s:
        x = torch.where(_from_words(s["allowed"], v), x, -torch.inf)
    best = torch.where(x == x.amax(-1, keepdim=True), torch.arange(v, device="cuda", dtype=torch.int32), v).amin(-1)
    return dict(logits=x, best=best)


def _token_bytes(case, place):
    """Places of a token's bytes in its page: K row, K norm, V row in its own order, V norm.  place: [...] -> [..., bytes]."""
    d = case["d"]
    pdk, pdv = d * case["kb"] // 8, d * case["vb"] // 8
    p = place[..., None]
    i, two = torch.arange(pdv, device="cuda"), torch.arange(2, device="cuda")
    i = torch.where(p & 2 != 0, (i + pdv // 2) % pdv, i)
    kn = PAGE * pdk
    return torch.cat([p * pdk + torch.arange(pdk, device="cuda"), kn + 2 * p + two, kn + 2 * PAGE + p * pdv + i,
                      kn + 2 * PAGE + PAGE * pdv + 2 * p + two], -1)


def _plain_commit(s):
    case, parents, tokens, nxt, pool = s["case"], s["parents"].long(), s["tokens"], s["nxt"], s["pool"]
    b, t = parents.shape
    idx = torch.arange(t, device="cuda")
    # a node is chosen by its parent if its token is the target's next one there and no sibling before it has it too
    fits = (parents >= 0) & (tokens == nxt.gather(1, parents.clamp(min=0)))
    twin = (parents[:, :, None] == parents[:, None, :]) & fits[:, None, :] & (idx[None, :] < idx[:, None])
    chosen = (fits & ~twin.any(-1)) | (idx == 0)
    reach = _reach(parents)
    on_path = ~(reach & ~chosen[:, None, :]).any(-1) & reach[:, :, 0]
    n = on_path.sum(-1)
    path = torch.where(on_path, idx, t).sort(-1).values
    live = idx < n[:, None]
    path = torch.where(live, path, -1)
    said = torch.where(live, nxt.gather(1, path.clamp(min=0)), -1)
    # the tokens of the path move behind the context
    ctx = s["lens"].long()[:, None] - t
    layers, nb, h, size = pool.shape

    def where(pos):   # [B, T] positions -> [L, B, T, H, bytes] places in the pool
        blk = s["table"].long().gather(1, pos // PAGE)
        row = (torch.arange(layers, device="cuda")[:, None, None] * nb + blk) * h
        row = row[..., None] + torch.arange(h, device="cuda")
        return row[..., None] * size + _token_bytes(case, pos % PAGE)[None, :, :, None]

    flat = pool.view(-1)
    src, dst = where(ctx + torch.where(live, path, idx)), where(ctx + idx)
    move = (live & (path != idx))[None, :, :, None, None].expand_as(src)
    flat[dst[move]] = flat[src[move]]
    return dict(path=path.to(torch.int32), accepted=n.to(torch.int32), tokens=said, seq_lens=(s["lens"] - t + n).to(torch.int32), pool=pool)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, t = case["kind"], case["tree"]
    if kind == "pages":
        ctx = _contexts(case)
        r, lens = len(ctx), ctx + t
        again = int((lens if case["packed"] else lens - ctx).sum())
        pages = again // PAGE + r
        tokens = again if case["packed"] else r * t
        # lengths in and out, four words for each page that comes and goes, slots, parents, masks, positions
        return dict(bytes=6 * 4 * r + 4 * 4 * pages + 8 * tokens + 4 * r * t * (2 + (t + 31) // 32), flops=0)
    if kind == "logits":
        r, v, es = case["requests"], case["vocab"], DTYPES[case["dtype"]].itemsize
        n = r * t * v
        said = int(_spread(r, case["history"], max(1, case["history"] // 16)).sum())
        return dict(bytes=n * (es + 4) + (n // 8 if case["grammar"] else 0) + 4 * said + 8 * r * case["biases"] + 4 * r * t, flops=2 * n)
    token = case["d"] * (case["kb"] + case["vb"]) // 8 + 4
    if kind == "commit":
        taken = _accepted(case)
        moved = int((taken & (taken.cumsum(-1) - 1 != torch.arange(t))).sum())
        return dict(bytes=2 * case["layers"] * case["hkv"] * moved * token + 20 * case["batch"] * t, flops=0)
    trees = _tree_lens(case)
    lens = _contexts(case) + trees
    es, d = DTYPES[case["dtype"]].itemsize, case["d"]
    # of the tree itself a node attends some nodes only: those products are left out
    return dict(bytes=int(lens.sum()) * case["hkv"] * token + 4 * int(((lens + 15) // 16).sum()) + 2 * case["batch"] * t * case["hq"] * d * es
                + 4 * case["batch"] * t * ((t + 31) // 32),
                flops=4.0 * case["hq"] * d * int((trees * (lens - trees)).sum()))


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    if case["kind"] in ("pages", "commit"):
        return None                       # whole numbers and bytes
    s = prepare(case, seed)
    if case["kind"] == "logits":
        r, t, v = s["logits"].shape
        x = s["logits"].double()
        for i in range(r):
            n, p = int(s["lens"][i]), int(s["prompt_lens"][i])
            prompt, answer = s["history"][i, :p].long(), s["history"][i, p:n].long()
            rep, freq, pres = (float(s[k][i]) for k in ("repetition", "frequency", "presence"))
            for j in range(t):
                path = _from_words(s["masks"][i, j], t).nonzero()[:, 0]
                c = torch.bincount(torch.cat([answer, s["tokens"][i, path].long()]), minlength=v).double()
                hit = c > 0
                hit[prompt] = True
                y = x[i, j]
                y = torch.where(hit, torch.where(y > 0, y / rep, y * rep), y) - freq * c - pres * (c > 0)
                if "bias" in s:
                    k = s["bias_ids"][i] >= 0
                    y = y.index_add(0, s["bias_ids"][i][k].long(), s["bias"][i][k].double())
                if "allowed" in s:
                    w = s["allowed"][i, j].long()
                    y[((w[torch.arange(v, device="cuda") // 32] >> (torch.arange(v, device="cuda") % 32)) & 1) == 0] = -torch.inf
                x[i, j] = y
        return dict(logits=x, best=None)
    d, h, t = case["d"], case["hkv"], case["tree"]
    g = case["hq"] // h
    had = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    while len(had) < d:
        had = torch.cat([torch.cat([had, had], 1), torch.cat([had, -had], 1)])
    rot = s["signs"].double()[:, None] * had / math.sqrt(d)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    widths = dict(k=(0, case["kb"]), v=(PAGE * (d * case["kb"] // 8 + 2), case["vb"]))

    def vectors(pages, which):
        at, bits = widths[which]
        pd = d * bits // 8
        stream = (pages[:, at:at + PAGE * pd].reshape(-1, pd, 1) >> torch.arange(8, device="cuda", dtype=torch.uint8)) & 1
        code = (stream.reshape(-1, d, bits).long() * 2 ** torch.arange(bits, device="cuda")).sum(-1)
        norm = pages[:, at + PAGE * pd:at + PAGE * (pd + 2)].contiguous().view(torch.float16).reshape(-1, 1).double()
        x = s["levels_" + which].double()[code] * norm
        if which == "v":
            place = torch.arange(len(x), device="cuda") % PAGE
            x = torch.where((place // 2 % 2 == 1)[:, None], x.roll(d // 2, 1), x)
        return x

    for i in range(case["batch"]):
        n, nodes = int(s["lens"][i]), int(s["tree_lens"][i])
        ids = s["table"][i, :(n + PAGE - 1) // PAGE].long()
        see = torch.ones(nodes, n, dtype=torch.bool, device="cuda")
        see[:, n - nodes:] = _from_words(s["masks"][i], t)[:nodes, :nodes]
        for j in range(h):
            k, v = (vectors(s["pages"][ids, j], w)[:n] for w in "kv")
            for e in range(g):
                q = s["q"][i, :nodes, j * g + e].double() @ rot
                p = torch.softmax((q @ k.T / math.sqrt(d)).masked_fill(~see, -torch.inf), -1)
                out[i, :nodes, j * g + e] = (p @ v) @ rot.T
    return dict(out=out)
