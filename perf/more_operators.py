"""Operators of beam search and parallel sampling on the compressed paged cache, measured against their plain forms.

A serving engine that keeps several candidate answers (beams, samples) of a prompt does this in a step: the best
continuations of every request's beams are chosen among all beams and the vocabulary, the beams' rows of the page table
become copies of those that they go on from (blocks are shared, only a partly filled last one is copied), and the next
token of every beam attends its cache, whose leading blocks are the same for all beams of a request.  From time to time
the blocks in use are moved together.  Four operators, one kind of case each:

  select     beam.select: the best continuations over beams and vocabulary, and what it would score to end
  fork       PageTable.fork + PagedKVPool.copy_pages + PageTable.shared_lens: rows become copies of others
  compact    PageTable.compact + PagedKVPool.copy_pages: blocks in use move to the lowest ids
  attention  PagedKVPool.shared_attention over one layer of the pool: one new token of every beam

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
        # one request of four beams on a local machine
        dict(name="select_single", kind="select", requests=1, beams=4, vocab=32768, best=4, ends=1, first=False, dtype="bf16"),
        # the first step of a mixed batch: only one beam of each request is alive; fp32 logits, rows of an odd length
        dict(name="select_first", kind="select", requests=24, beams=5, vocab=50257, best=5, ends=1, first=True, dtype="fp32"),
        # a serving batch, twice as many candidates as beams
        dict(name="select_serving", kind="select", requests=64, beams=8, vocab=131072, best=16, ends=2, first=False, dtype="bf16"),
        # one request's four beams go on, the caches of all layers
        dict(name="fork_single", kind="fork", requests=1, beams=4, ctx=900, own=40, cut=False, hkv=8, d=128, kb=4, vb=4, layers=32),
        # a serving batch of beams
        dict(name="fork_serving", kind="fork", requests=32, beams=8, ctx=600, own=150, cut=False, hkv=8, d=128, kb=4, vb=4, layers=32),
        # a small cache after half of its requests have ended
        dict(name="compact_small", kind="compact", requests=24, ctx=900, hkv=2, d=64, kb=3, vb=3, layers=24),
        # a serving cache, all layers
        dict(name="compact_serving", kind="compact", requests=96, ctx=1200, hkv=8, d=128, kb=4, vb=3, layers=32),
        # one request of four beams: every microsecond shows
        dict(name="attention_single", kind="attention", requests=1, beams=4, ctx=900, own=40, ragged=False, hq=32, hkv=8,
             d=128, kb=4, vb=4, dtype="bf16"),
        # a serving batch of beams over long prompts
        dict(name="attention_serving", kind="attention", requests=32, beams=8, ctx=8192, own=128, ragged=False, hq=32,
             hkv=8, d=128, kb=4, vb=4, dtype="bf16"),
        # a small model's mixed batch of five samples each, 3-bit codes, some samples ended
        dict(name="attention_small_model", kind="attention", requests=40, beams=5, ctx=4096, own=300, ragged=True, hq=14,
             hkv=2, d=64, kb=3, vb=3, dtype="fp16"),
        # heads of 256 with 2-bit values, a mixed batch
        dict(name="attention_wide_heads", kind="attention", requests=24, beams=4, ctx=16384, own=200, ragged=True, hq=16,
             hkv=8, d=256, kb=4, vb=2, dtype="bf16"),
        # long documents, GQA group 8
        dict(name="attention_long", kind="attention", requests=4, beams=4, ctx=65536, own=400, ragged=False, hq=64, hkv=8,
             d=128, kb=3, vb=3, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["select", "select", "fork", "compact", "attention", "attention", "attention"])
    beams = rng.choice([1, 2, 3, 4, 4, 5, 8, 8, 12, 16])
    if kind == "select":
        vocab = _log_int(rng, 1000, 160000)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        requests = _log_int(rng, 1, max(1, min(256, (1 << 27) // (vocab * beams * DTYPES[dtype].itemsize))))
        return dict(kind=kind, requests=requests, beams=beams, vocab=vocab, best=_log_int(rng, 1, 32), ends=rng.choice([0, 1, 2, 5]),
                    first=rng.random() < 0.2, dtype=dtype)
    d, hkv = rng.choice([64, 128, 128, 128, 256]), rng.choice([1, 2, 4, 8])
    kb, vb = rng.choice([2, 3, 4, 4]), rng.choice([2, 3, 4, 4])
    if kind == "attention":
        group = rng.choice([1, 2, 4, 4, 7, 8, 16])
        requests = _log_int(rng, 1, 64)
        # tokens x heads of the cache and products of a pass stay below those of the longest listed cases
        top = min(65536, (1 << 28) // (d * requests * hkv), (1 << 33) // (d * requests * hkv * group * beams))
        return dict(kind=kind, requests=requests, beams=beams, ctx=_log_int(rng, 1, max(64, top)),
                    own=_log_int(rng, 1, max(1, min(600, (1 << 25) // (d * requests * beams * hkv), (1 << 31) // (d * requests * hkv * group * beams)))), ragged=rng.random() < 0.4,
                    hq=hkv * group, hkv=hkv, d=d, kb=kb, vb=vb, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    # blocks x heads x layers stay below those of the longest listed case
    layers = _log_int(rng, 1, 48)
    blocks = (1 << 26) // (layers * hkv * d)
    if kind == "compact":
        requests = _log_int(rng, 2, max(2, min(256, blocks // 4)))
        return dict(kind=kind, requests=requests, ctx=_log_int(rng, 1, max(1, min(2000, 8 * blocks // requests))), hkv=hkv, d=d, kb=kb,
                    vb=vb, layers=layers)
    requests = _log_int(rng, 1, max(1, min(64, blocks // (16 * beams))))
    return dict(kind=kind, requests=requests, beams=beams, ctx=_log_int(rng, 1, 600), own=_log_int(rng, 1, 150), cut=rng.random() < 0.4,
                hkv=hkv, d=d, kb=kb, vb=vb, layers=layers)


# ------------------------------------------------------------------ what a case is made of
def _spread(n, top, low):
    """n lengths, log-uniform in [low, top], the first the longest: a fixed mix, the same work for every seed."""
    u = torch.rand(n, generator=torch.Generator("cpu").manual_seed(20250))
    x = torch.exp(math.log(low) + u * (math.log(top) - math.log(low))).to(torch.int64).clamp(low, top)
    x[0] = top
    return x


def _lengths(case):
    """(tokens of the prompts [R], tokens of all rows [R * K]): beams of a request are equally long, of a mixed batch's
    samples one in nine has ended."""
    r, k = case["requests"], case["beams"]
    if not case.get("ragged"):
        ctx, own = torch.full((r,), case["ctx"]), torch.full((r,), case["own"])
    else:
        ctx, own = _spread(r, case["ctx"], max(1, case["ctx"] // 256)), _spread(r, case["own"], max(1, case["own"] // 32)).flip(0)
    lens = (ctx + own).repeat_interleave(k)
    if case.get("ragged"):
        lens[torch.arange(r * k) % 9 == 5] = 0
    return ctx, lens


def _shared_table(case, gen):
    """Block table of the rows (a prompt's whole blocks are the same for its rows), their lengths, shared tokens and the number
    of blocks; ids are shuffled."""
    k = case["beams"]
    ctx, lens = _lengths(case)
    both = (ctx // PAGE)
    per = (lens + PAGE - 1) // PAGE
    rest = (per - both.repeat_interleave(k)).clamp(min=0)
    live = lens.view(-1, k).amax(1) > 0
    nb = int((both * live).sum() + rest.sum())
    width = max(1, int(per.max()))
    ids = torch.randperm(nb, device="cuda", generator=gen).to(torch.int32)
    col = torch.arange(width)
    at_both = torch.cat([torch.zeros(1, dtype=torch.int64), (both * live).cumsum(0)])
    at_rest = at_both[-1] + torch.cat([torch.zeros(1, dtype=torch.int64), rest.cumsum(0)])
    first = both.repeat_interleave(k)[:, None]
    place = torch.where(col < first, at_both[:-1].repeat_interleave(k)[:, None] + col, at_rest[:-1][:, None] + col - first)
    held = (col < per[:, None]).cuda()
    table = torch.where(held, ids[torch.where(col < per[:, None], place, 0).cuda()], -1)
    return table, lens, (both * PAGE * live), nb


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
    return {"select": _prepare_select, "fork": _prepare_fork, "compact": _prepare_compact,
            "attention": _prepare_attention}[case["kind"]](case, gen)


def _prepare_select(case, gen):
    r, k, v = case["requests"], case["beams"], case["vocab"]
    logits = (2.5 * torch.randn(r, k, v, device="cuda", generator=gen)).to(DTYPES[case["dtype"]])
    scores = -3 * torch.rand(r, k, device="cuda", generator=gen)
    scores = scores.cumsum(1) - 40 * torch.rand(r, 1, device="cuda", generator=gen)
    if case["first"]:
        scores[:, 0], scores[:, 1:] = 0, -torch.inf
    ends = None
    if case["ends"]:    # what ends an answer is likely now and then
        ends = torch.randperm(v, device="cuda", generator=gen)[:case["ends"]].to(torch.int32)
        logits[..., ends.long()] += 3 * torch.randn(r, k, case["ends"], device="cuda", generator=gen).to(logits.dtype)
    return dict(case=case, logits=logits, scores=scores, ends=ends)


def _handle(pool, case):
    from fused_turboquant_b200 import PagedKVPool
    h = PagedKVPool(pool.shape[1], case["hkv"], case["d"], case["kb"], case["vb"], n_layers=len(pool), seed=SIGN_SEED,
                    device="cuda")
    h.pool.copy_(pool)
    return h


def _bytes(case, nb, gen):
    """Pages whose contents do not matter."""
    size = PAGE * (case["d"] * (case["kb"] + case["vb"]) // 8 + 4)
    return torch.randint(-(1 << 31), 1 << 31, (case["layers"], nb, case["hkv"], size // 4), dtype=torch.int32, device="cuda",
                         generator=gen).view(torch.uint8)


def _table_state(s, case, state):
    if own:   # the handle that an engine keeps
        from fused_turboquant_b200 import PageTable
        s["pages"] = PageTable(len(state["free_blocks"]), len(state["seq_lens"]), state["block_table"].shape[1], device="cuda",
                               sharing="shares" in state)
        s["pages"].load_state_dict(state)
        s["pool"] = _handle(s["pool"], case)
    else:
        s["table"] = state
    return s


def _prepare_fork(case, gen):
    """Beams that share their prompt's blocks, and who goes on from whom; with `cut` samples that are cut back and ended too."""
    r, k = case["requests"], case["beams"]
    table, lens, _, nb = _shared_table(case, gen)
    spare = 2 * r * k + nb // 8
    free = torch.full((nb + spare,), -1, dtype=torch.int32, device="cuda")
    free[:spare] = nb + torch.randperm(spare, device="cuda", generator=gen).to(torch.int32)
    held = torch.bincount(table[table >= 0].long(), minlength=nb + spare)
    state = dict(block_table=table, seq_lens=lens.to("cuda", torch.int32), free_blocks=free,
                 n_free=torch.tensor([spare], dtype=torch.int32, device="cuda"), shares=(held - 1).clamp(min=0).to(torch.int32))
    s = dict(case=case, parents=torch.randint(0, k, (r, k), device="cuda", generator=gen).to(torch.int32), keep=None)
    if case["cut"]:
        u = torch.rand(r, k, device="cuda", generator=gen)
        s["parents"] = torch.where(u < 0.2, -1, torch.where(u < 0.6, torch.arange(k, device="cuda"), s["parents"])).to(torch.int32)
        s["keep"] = (lens.cuda() * torch.rand(r * k, device="cuda", generator=gen).sqrt()).to(torch.int32)
    s["pool"] = _bytes(case, nb + spare, gen)
    return _table_state(s, case, state)


def _prepare_compact(case, gen):
    """A cache that was full; half of its requests have ended, and their blocks came free in any order."""
    r = case["requests"]
    lens = _spread(r, case["ctx"], max(1, case["ctx"] // 8))
    per = (lens + PAGE - 1) // PAGE
    nb, width = int(per.sum()), int(per.max())
    ids = torch.randperm(nb, device="cuda", generator=gen).to(torch.int32)
    col = torch.arange(width, device="cuda")
    stays = (torch.arange(r) % 2 == 0).cuda()
    start = (per.cumsum(0) - per).cuda()
    held = col < per.cuda()[:, None]
    full = torch.where(held, ids[torch.where(held, start[:, None] + col, 0)], -1)
    table = torch.where(stays[:, None], full, -1)
    gone = full[(~stays)[:, None] & held]
    free = torch.full((nb,), -1, dtype=torch.int32, device="cuda")
    free[:len(gone)] = gone
    s = dict(case=case, fragmented=dict(block_table=table, seq_lens=torch.where(stays, lens.cuda(), 0).to(torch.int32), free_blocks=free,
                                        n_free=torch.tensor([len(gone)], dtype=torch.int32, device="cuda")))
    s["pool"] = _bytes(case, nb, gen)
    return _table_state(s, case, {k: v.clone() for k, v in s["fragmented"].items()})


def _prepare_attention(case, gen):
    d, b = case["d"], case["requests"] * case["beams"]
    table, lens, shared, nb = _shared_table(case, gen)
    pool = _pool(1, nb, case["hkv"], d, case["kb"], case["vb"], gen)
    s = dict(case=case, table=table, lens=lens.to("cuda", torch.int32), shared=shared.to("cuda", torch.int32), top=int(lens.max()),
             on_host=lens.tolist(), q=torch.randn(b, case["hq"], d, device="cuda", generator=gen).to(DTYPES[case["dtype"]]))
    s.update(pages=pool[0], signs=_signs(d), hadamard=_hadamard(d),
             levels_k=torch.from_numpy(_codebook(d, case["kb"])[0]).cuda(), levels_v=torch.from_numpy(_codebook(d, case["vb"])[0]).cuda())
    if own:
        s["pool"] = _handle(pool, case)
    return s


# ------------------------------------------------------------------ a pass
def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if not own:
        return {"select": _plain_select, "fork": _plain_fork, "compact": _plain_compact, "attention": _plain_attention}[kind](s)
    from fused_turboquant_b200 import beam
    if kind == "select":
        got = beam.select(s["logits"], s["scores"], case["best"], end_tokens=s["ends"])
        return dict(scores=got.scores, parents=got.parents, tokens=got.tokens, end_scores=got.end_scores)
    if kind == "attention":
        return dict(out=s["pool"].shared_attention(s["q"], s["table"], s["lens"], s["top"], s["shared"]))
    p, pool = s["pages"], s["pool"]
    if kind == "fork":
        got = p.fork(s["parents"], keep_lens=s["keep"])
        pool.copy_pages(got.copies)
        return dict(copies=got.copies, done=got.done, shared=p.shared_lens(case["beams"]), pool=pool.pool, **p.state_dict())
    p.load_state_dict(s["fragmented"])
    copies = p.compact()
    pool.copy_pages(copies)
    return dict(copies=copies, pool=pool.pool, **p.state_dict())


def _plain_select(s):
    x = s["logits"].double()
    r, k, v = x.shape
    best = s["case"]["best"]
    x = x - x.amax(-1, keepdim=True)
    x = x - torch.log(torch.exp(x).sum(-1, keepdim=True)) + s["scores"].double()[..., None]
    x = torch.where(torch.isnan(x), -torch.inf, x)
    ends = None
    if s["ends"] is not None:
        ends = x[..., s["ends"].long()].float()
        x[..., s["ends"].long()] = -torch.inf
    x = x.view(r, k * v)
    n = min(best, k * v)
    scores, at = [], []
    for _ in range(n):      # the largest, the first of equal ones
        m = x.amax(-1, keepdim=True)
        i = torch.where(x == m, torch.arange(k * v, device="cuda"), k * v).amin(-1, keepdim=True)
        x.scatter_(1, i, -torch.inf)
        scores.append(m)
        at.append(i)
    scores, at = torch.cat(scores, 1), torch.cat(at, 1)
    none = scores == -torch.inf
    pad = (0, best - n)
    fill = torch.nn.functional.pad
    return dict(scores=fill(scores.float(), pad, value=-math.inf), parents=fill(torch.where(none, -1, at // v), pad, value=-1).to(torch.int32),
                tokens=fill(torch.where(none, -1, at % v), pad, value=-1).to(torch.int32), end_scores=ends)


def _copy(pool, copies):
    live = (copies >= 0).all(1)
    pool[:, copies[live, 1].long()] = pool[:, copies[live, 0].long()]


def _shared(table, lens, k):
    """Leading tokens in whole blocks that all rows of a group have in common; rows without tokens do not count."""
    t, n = table.view(-1, k, table.shape[1]), lens.view(-1, k)
    live = n > 0
    first = t.gather(1, live.int().argmax(1)[:, None, None].expand(-1, 1, t.shape[2]))
    whole = torch.arange(t.shape[2], device="cuda") < (n // PAGE)[..., None]
    same = (((t == first) & whole) | ~live[..., None]).all(1) & live.any(1)[:, None]
    return PAGE * same.int().cumprod(1).sum(1).to(torch.int32)


def _plain_fork(s):
    st, case = s["table"], s["case"]
    table, lens, free, n_free, shares = (st[n] for n in ("block_table", "seq_lens", "free_blocks", "n_free", "shares"))
    n, width = table.shape
    k, nb = case["beams"], len(free)
    row, col = torch.arange(n, device="cuda"), torch.arange(width, device="cuda")
    par = s["parents"].long()
    ok = ((par >= 0) & (par < k)).view(-1)
    par = (par.clamp(0, k - 1) + k * torch.arange(len(par), device="cuda")[:, None]).view(-1)
    new_lens = torch.where(ok, lens[par], 0)
    if s["keep"] is not None:
        new_lens = torch.minimum(new_lens, s["keep"].clamp(min=0))
    pages = (new_lens + PAGE - 1) // PAGE
    new = torch.where(col < pages[:, None], table[par], -1)

    def count(ids, weight=None):
        return torch.zeros(nb, dtype=torch.int64, device="cuda").index_add_(0, ids, torch.ones_like(ids) if weight is None else weight)

    held = count(new[new >= 0].long())
    # a partly filled last block that several rows would hold: the first of them keeps it, unless it is another row's whole one
    last = new.gather(1, (pages - 1).clamp(min=0)[:, None].long())[:, 0].clamp(min=0).long()
    part = new_lens % PAGE != 0
    parts = count(last, part.long())
    keeper = torch.full((nb,), n, device="cuda").scatter_reduce_(0, last, torch.where(part, row, n), "amin")
    need = part & (held[last] > 1) & ~((held[last] == parts[last]) & (keeper[last] == row))
    # blocks that nobody holds any more, in the order of the rows; the first of them lies on top
    old = table[(col < ((lens + PAGE - 1) // PAGE)[:, None])].long()
    at = torch.full((nb,), len(old), device="cuda").scatter_reduce_(0, old, torch.arange(len(old), device="cuda"), "amin")
    gone = old[(held[old] == 0) & (at[old] == torch.arange(len(old), device="cuda"))]
    copies = torch.full((n, 2), -1, dtype=torch.int32, device="cuda")
    wanted = int(need.sum())
    done = wanted <= int(n_free) + len(gone)
    if done:
        top = n_free + len(gone)
        free[top - 1 - torch.arange(len(gone), device="cuda")] = gone.to(torch.int32)
        taken = free[top - 1 - torch.arange(wanted, device="cuda")]
        copies[:wanted, 0], copies[:wanted, 1] = last[need].to(torch.int32), taken
        new[need, (pages - 1)[need].long()] = taken
        n_free.copy_(top - wanted)
        table.copy_(new)
        lens.copy_(new_lens)
        shares.copy_((count(new[new >= 0].long()) - 1).clamp(min=0))
    _copy(s["pool"], copies)
    return dict(copies=copies, done=torch.tensor([done], dtype=torch.int32, device="cuda"), shared=_shared(table, lens, k), pool=s["pool"], **st)


def _plain_compact(s):
    st = s["table"]
    for name, x in s["fragmented"].items():
        st[name].copy_(x)
    table, free = st["block_table"], st["free_blocks"]
    nb, n = len(free), int(st["n_free"])
    used = torch.ones(nb, dtype=torch.bool, device="cuda")
    used[free[:n].long()] = False
    # the lowest block in use behind the first nb - n goes to the lowest hole before that, and so on
    holes, movers = (~used[:nb - n]).nonzero()[:, 0], used[nb - n:].nonzero()[:, 0] + nb - n
    to = torch.arange(nb, device="cuda")
    to[movers] = holes
    copies = torch.full((nb // 2, 2), -1, dtype=torch.int32, device="cuda")
    copies[:len(holes), 0], copies[:len(holes), 1] = movers.to(torch.int32), holes.to(torch.int32)
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    free[:n] = nb - 1 - torch.arange(n, device="cuda", dtype=torch.int32)
    _copy(s["pool"], copies)
    return dict(copies=copies, pool=s["pool"], **st)


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
    b, hq, d = s["q"].shape
    h, pdk, pdv = case["hkv"], d * case["kb"] // 8, d * case["vb"] // 8
    q = (s["q"].float() * s["signs"]) @ s["hadamard"] / math.sqrt(d)
    out = torch.zeros(b, h, hq // h, d, device="cuda")
    odd = (torch.arange(PAGE, device="cuda") & 2 != 0)[:, None]

    def dense(rows, norms, levels, bits, width, n):
        x = levels[_unpack(rows.reshape(h, -1, PAGE, width), bits).int()]
        if levels is s["levels_v"]:
            x = torch.where(odd, torch.cat([x[..., d // 2:], x[..., :d // 2]], -1), x)
        x = x * norms.contiguous().view(torch.float16).float()[..., None]
        return x.flatten(1, 2)[:, :n]                                               # [H, n, D]

    for i, n in enumerate(s["on_host"]):        # a row at a time: its keys and values would not fit otherwise
        if n == 0:
            continue
        pages = s["pages"][s["table"][i, :(n + PAGE - 1) // PAGE].long()].transpose(0, 1)       # [H, blocks, bytes]
        k, kn, v, vn = pages.split([PAGE * pdk, 2 * PAGE, PAGE * pdv, 2 * PAGE], -1)
        w = q[i].view(h, hq // h, d) @ dense(k, kn, s["levels_k"], case["kb"], pdk, n).transpose(-1, -2) * d ** -0.5
        w = torch.exp(w - w.amax(-1, keepdim=True))
        out[i] = w @ dense(v, vn, s["levels_v"], case["vb"], pdv, n) / w.sum(-1, keepdim=True)
    out = (out.view(b, hq, d) @ s["hadamard"] / math.sqrt(d)) * s["signs"]
    return dict(out=out.to(s["q"].dtype))


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "select":
        rows = case["requests"] * case["beams"]
        alive = case["requests"] if case["first"] else rows       # what a dead beam's logits are does not matter
        return dict(bytes=alive * case["vocab"] * DTYPES[case["dtype"]].itemsize + 4 * rows * (1 + case["ends"]) + 12 * case["requests"] * case["best"],
                    flops=3 * alive * case["vocab"])
    token = case["d"] * (case["kb"] + case["vb"]) // 8 + 4
    if kind == "compact":
        lens = _spread(case["requests"], case["ctx"], max(1, case["ctx"] // 8))
        per = (lens + PAGE - 1) // PAGE
        nb, n = int(per.sum()), int(per[1::2].sum())
        moved = n * (nb - n) / nb           # blocks in use behind the first nb - n, of shuffled ids
        return dict(bytes=2 * moved * PAGE * token * case["hkv"] * case["layers"] + 8 * (nb - n) + 8 * n + 8 * moved, flops=0)
    ctx, lens = _lengths(case)
    r, k = case["requests"], case["beams"]
    per = (lens + PAGE - 1) // PAGE
    if kind == "fork":
        # of k beams that go on from any of k, the expected number that cannot keep the block of the one they go on from
        copied = r * (k - k * (1 - (1 - 1 / k) ** k)) if int(lens[0]) % PAGE else 0
        if case["cut"]:
            copied = 0.4 * copied
        own_pages = int((per - (ctx // PAGE).repeat_interleave(k)).sum())
        return dict(bytes=2 * copied * token * PAGE * case["hkv"] * case["layers"] + 8 * own_pages + 16 * r * k, flops=0)
    es, d = DTYPES[case["dtype"]].itemsize, case["d"]
    own_tokens = int((lens - (ctx // PAGE * PAGE).repeat_interleave(k)).clamp(min=0).sum())
    tokens = own_tokens + int((ctx // PAGE * PAGE).sum())
    return dict(bytes=tokens * case["hkv"] * token + 4 * (tokens // PAGE) + 2 * r * k * case["hq"] * d * es,
                flops=4.0 * case["hq"] * d * int(lens.sum()))


# ------------------------------------------------------------------ from the definitions, in 64 bits
def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None                       # whole numbers and bytes
    s = prepare(case, seed)
    if case["kind"] == "select":
        r, k, v = s["logits"].shape
        best = case["best"]
        scores = torch.full((r, best), -math.inf, dtype=torch.float64, device="cuda")
        ends = None if s["ends"] is None else torch.empty(r, k, case["ends"], dtype=torch.float64, device="cuda")
        for i in range(r):
            x = torch.log_softmax(s["logits"][i].double(), -1) + s["scores"][i].double()[:, None]
            if ends is not None:
                ends[i] = x[:, s["ends"].long()]
                x[:, s["ends"].long()] = -math.inf
            top = x.flatten().sort(descending=True).values[:best]
            scores[i, :len(top)] = top
        return dict(scores=scores, parents=None, tokens=None, end_scores=ends)
    d, h, k = case["d"], case["hkv"], case["beams"]
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

    shared = s["shared"].tolist()
    for r in range(case["requests"]):
        rows = [i for i in range(r * k, r * k + k) if s["on_host"][i] > 0]
        for j in range(h):
            front = {}
            for i in rows:
                n, cut = s["on_host"][i], shared[r] // PAGE
                ids = s["table"][i, :(n + PAGE - 1) // PAGE].long()
                if not front:       # (the same blocks for all of them)
                    front = {w: vectors(s["pages"][ids[:cut], j], w) for w in "kv"}
                key, val = (torch.cat([front[w], vectors(s["pages"][ids[cut:], j], w)])[:n] for w in "kv")
                p = torch.softmax(s["q"][i, j * g:j * g + g].double() @ rot @ key.T / math.sqrt(d), -1)
                out[i, j * g:j * g + g] = (p @ val) @ rot.T
    return dict(out=out)
