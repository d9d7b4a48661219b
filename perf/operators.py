"""Measured cases of the serving operators around masked selection: filtered sampling, page planning, rotary
append into a paged cache, and attention of a chunk of new tokens over that cache.

One decoding round uses them in this order: ``plan_pages`` brings the block tables to the round's lengths, every
layer rotates and appends its new keys and values (``rotary_append``) and attends over the cache
(``chunk_attention``), and ``batched_filtered_sample`` draws each row's token under its grammar mask.

``run`` computes an operator in elementary torch operations, or, with ``own`` set, through this repository's entry
points.  Cases are plain dicts; ragged lengths are drawn from the case's own ``lens`` seed, values from ``prepare``'s.
"""

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 1 << 27  # elements of the plain forms' largest temporaries


def listed():
    """The measured cases."""
    return [
        # The eight fp16 rows of the sampling configuration, as one small decode step draws them: latency.
        dict(name="sample-decode8-topk", op="sample", rows=8, vocab=248320, dtype="float16", filters="top_k", dense=True, lens=1),
        # A full decode batch whose requests bring their own temperature and filters, grammar masks of every density.
        dict(name="sample-batch256-mixed", op="sample", rows=256, vocab=151936, dtype="bfloat16", filters="mixed", dense=False, lens=2),
        # A vocabulary whose rows start on odd addresses, float32 scores, free text with min-p.
        dict(name="sample-odd64-minp", op="sample", rows=64, vocab=50257, dtype="float32", filters="min_p", dense=True, lens=3),
        # The target rows of a verification round (K + 1 = 9 per sequence) sampled with nucleus filtering: the largest.
        dict(name="sample-verify1152-topp", op="sample", rows=1152, vocab=248320, dtype="bfloat16", filters="top_p", dense=False, lens=4),
        # Page bookkeeping of a small decode batch, one drafted window per sequence.
        dict(name="plan-round32", op="plan", seqs=32, new_lo=1, new_hi=9, past_lo=0, past_hi=2000, page=16, lens=5),
        # A large batch that admits prompts, drops finished requests and rolls drafts back.
        dict(name="plan-admit1024", op="plan", seqs=1024, new_lo=0, new_hi=256, past_lo=0, past_hi=8000, page=32, lens=6),
        # One verification window of the end-to-end target (16 heads of 64, 4 shared key heads).
        dict(name="append-round8", op="append", seqs=8, new_lo=9, new_hi=9, past_lo=10, past_hi=500, heads=16, kv_heads=4, dim=64,
             page=16, dtype="bfloat16", lens=7),
        # Prompts packed into one step.
        dict(name="append-prompts", op="append", seqs=24, new_lo=100, new_hi=1500, past_lo=0, past_hi=4000, heads=32, kv_heads=8, dim=128,
             page=64, dtype="float16", lens=8),
        # Single-token decode of the end-to-end target: short caches, latency.
        dict(name="attend-decode8", op="attend", seqs=8, new_lo=1, new_hi=1, past_lo=64, past_hi=600, heads=16, kv_heads=4, dim=64,
             page=16, window=0, sinks=0, dtype="bfloat16", lens=9),
        # A verification round: nine rows per sequence over long ragged caches, bound by reading keys and values.
        dict(name="attend-verify64", op="attend", seqs=64, new_lo=9, new_hi=9, past_lo=500, past_hi=12000, heads=32, kv_heads=8, dim=128,
             page=32, window=0, sinks=0, dtype="bfloat16", lens=10),
        # Prompt chunks over what earlier chunks left in the cache: bound by the products.
        dict(name="attend-chunks4", op="attend", seqs=4, new_lo=1500, new_hi=2500, past_lo=0, past_hi=12000, heads=32, kv_heads=8, dim=128,
             page=64, window=0, sinks=0, dtype="bfloat16", lens=11),
        # Long streams with a sliding window and four first tokens that stay visible.
        dict(name="attend-window16", op="attend", seqs=16, new_lo=1, new_hi=400, past_lo=3, past_hi=30000, heads=24, kv_heads=8, dim=64,
             page=16, window=1000, sinks=4, dtype="float16", lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges."""
    op = rng.choice(["sample", "sample", "plan", "append", "attend", "attend", "attend"])
    seed = rng.randrange(1 << 30)
    if op == "sample":
        vocab = rng.choice([248320, 151936, 50257, _log(rng, 1000, 248320), _log(rng, 1000, 248320)])
        rows = _log(rng, 1, min(1152, 60_000_000 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(list(DTYPES)), filters=rng.choice(["top_k", "top_p", "min_p", "mixed"]),
                    dense=rng.random() < 0.5, lens=seed)
    if op == "plan":
        return dict(op=op, seqs=_log(rng, 1, 1024), new_lo=rng.choice([0, 1]), new_hi=_log(rng, 1, 256), past_lo=0, past_hi=_log(rng, 10, 8000),
                    page=rng.choice([8, 16, 32, 64]), lens=seed)
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8])
    dim = rng.choice([64, 128])
    dtype = rng.choice(["bfloat16", "float16"])
    page = rng.choice([16, 32, 64, 128])
    new_hi = _log(rng, 1, 1500)
    new_lo = rng.choice([0, 1, new_hi])
    if op == "append":
        most = max(1, 860_000 // (new_hi * (heads + 2 * kv_heads)))
        return dict(op=op, seqs=_log(rng, 1, min(24, most)), new_lo=new_lo, new_hi=new_hi, past_lo=0, past_hi=_log(rng, 10, 4000), heads=heads,
                    kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, lens=seed)
    past_hi = _log(rng, 10, 12000)
    most = int(1e12 / (4 * new_hi * (past_hi + new_hi) * heads * dim))
    seqs = _log(rng, 1, max(1, min(64 if new_hi <= 16 else 4, most)))
    window = rng.choice([0, 0, _log(rng, 1, 4000)])
    return dict(op=op, seqs=seqs, new_lo=new_lo, new_hi=new_hi, past_lo=0, past_hi=past_hi, heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, window=window, sinks=rng.choice([0, 1, 4, 33]) if window else 0, dtype=dtype, lens=seed)


# ---------------------------------------------------------------- inputs
def _lengths(case):
    """(new tokens, tokens in the cache before them) of each sequence."""
    rng = random.Random(case["lens"])
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    past = [rng.randint(case["past_lo"], case["past_hi"]) for _ in range(case["seqs"])]
    if sum(new) == 0:
        new[0] = 1
    return new, past


def _prepare_sample(case, gen, dev):
    rows, vocab = case["rows"], case["vocab"]
    # Scores as a model gives them: a broad body, a few tokens well ahead of it, each row with its own sharpness.
    sharp = torch.rand((rows, 1), generator=gen, device=dev) * 2 + 1.5
    logits = torch.empty((rows, vocab), dtype=DTYPES[case["dtype"]], device=dev)
    words = (vocab + 31) // 32
    masks = torch.empty((rows, words), dtype=torch.int32, device=dev)
    density = torch.ones(rows, device=dev) if case["dense"] else torch.rand(rows, generator=gen, device=dev).mul(-7).exp()
    shifts = torch.arange(32, device=dev, dtype=torch.int64)
    step = max(1, BLOCK // (words * 32))
    for r0 in range(0, rows, step):
        n = min(step, rows - r0)
        x = torch.randn((n, vocab), generator=gen, device=dev) * sharp[r0:r0 + n]
        top = torch.randint(vocab, (n, 12), generator=gen, device=dev)
        x.scatter_add_(1, top, torch.rand((n, 12), generator=gen, device=dev) * 8)
        logits[r0:r0 + n] = x.to(logits.dtype)
        valid = torch.rand((n, words * 32), generator=gen, device=dev) < density[r0:r0 + n, None]
        valid.scatter_(1, top, True)
        for i in range(n):  # packed row by row to keep the temporaries small
            bits = (valid[i].view(words, 32).long() << shifts).sum(1)
            masks[r0 + i] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
    params = dict(temperature=0.7, top_k=0, top_p=1.0, min_p=0.0)
    if case["filters"] == "top_k":
        params.update(top_k=50, top_p=0.95)
    elif case["filters"] == "top_p":
        params.update(temperature=1.0, top_p=0.9)
    elif case["filters"] == "min_p":
        params.update(temperature=1.2, min_p=0.05)
    else:
        def pick(values, dtype):
            at = torch.randint(len(values), (rows,), generator=gen, device=dev)
            return torch.tensor(values, dtype=dtype, device=dev)[at]
        params = dict(temperature=pick([0.0, 0.6, 0.7, 0.8, 1.0, 1.0, 1.2], torch.float32),
                      top_k=pick([0, 0, 1, 20, 50, 1000, 5000], torch.int32),
                      top_p=pick([1.0, 1.0, 0.8, 0.9, 0.95], torch.float32), min_p=pick([0.0, 0.0, 0.02, 0.1], torch.float32))
    uniforms = torch.rand(rows, dtype=torch.float64, generator=gen, device=dev)
    return dict(case=case, logits=logits, masks=masks, uniforms=uniforms, params=params)


def _prepare_plan(case, gen, dev):
    new, past = _lengths(case)
    page = case["page"]
    rng = random.Random(case["lens"] + 1)
    # What each sequence holds from the step before: about its past, more after a rolled-back draft or an old request.
    held = [-(-p // page) + rng.choice([0, 0, 0, 1, 5]) for p in past]
    width = max(max(held), max(-(-(p + n) // page) for p, n in zip(past, new))) + 2
    used = sum(held)
    spare = sum(-(-n // page) + 1 for n in new)
    pages = used + spare + 7
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros((case["seqs"], width), dtype=torch.int32, device=dev)
    held_t = torch.tensor(held, dtype=torch.int32, device=dev)
    cell = torch.arange(width, device=dev)[None, :] < held_t[:, None]
    table[cell] = order[:used]
    free = torch.zeros(pages, dtype=torch.int32, device=dev)
    free[:pages - used] = order[used:]
    return dict(case=case, past=torch.tensor(past, dtype=torch.int32, device=dev), new=torch.tensor(new, dtype=torch.int32, device=dev),
                held=held_t, table=table, free=free, count=torch.tensor([pages - used], dtype=torch.int32, device=dev), tokens=sum(new))


def _prepare_cache(case, gen, dev):
    """A paged cache with every sequence's pages in it, in no order, and the step's lengths."""
    new, past = _lengths(case)
    page = case["page"]
    need = [-(-(p + n) // page) for p, n in zip(past, new)]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    width = max(1, max(need))
    cell = torch.arange(width, device=dev)[None, :] < torch.tensor(need, device=dev)[:, None]
    table = torch.zeros((case["seqs"], width), dtype=torch.int32, device=dev)
    table[cell] = order[:sum(need)]
    shape = (pages, page, case["kv_heads"], case["dim"])
    k = torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).to(DTYPES[case["dtype"]])
    v = torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).to(DTYPES[case["dtype"]])
    starts = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
    total = torch.tensor([p + n for p, n in zip(past, new)], dtype=torch.int32, device=dev)
    return dict(case=case, new=new, past=past, table=table, k=k, v=v, query_start=starts, seq_lens=total, tokens=sum(new))


def _prepare_append(case, gen, dev):
    state = _prepare_cache(case, gen, dev)
    n, heads, kv_heads, dim, page = state["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    # One projection's output holds queries, keys and values side by side: the operator gets strided views of it.
    fused = torch.randn((n, heads + 2 * kv_heads, dim), generator=gen, device=dev).to(DTYPES[case["dtype"]])
    state.update(q=fused[:, :heads], key=fused[:, heads:heads + kv_heads], value=fused[:, heads + kv_heads:])
    positions = torch.cat([torch.arange(p, p + m, device=dev) for p, m in zip(state["past"], state["new"])])
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device=dev), torch.tensor(state["new"], device=dev))
    state["positions"] = positions.to(torch.int32)
    state["slots"] = state["table"][seq, positions // page].long() * page + positions % page
    limit = max(p + m for p, m in zip(state["past"], state["new"]))
    inv = 1.0 / (1e6 ** (torch.arange(0, dim, 2, dtype=torch.float64, device=dev) / dim))
    angle = torch.arange(limit, dtype=torch.float64, device=dev)[:, None] * inv[None, :]
    state.update(cos=angle.cos().float(), sin=angle.sin().float())
    return state


def _prepare_attend(case, gen, dev):
    state = _prepare_cache(case, gen, dev)
    q = torch.randn((state["tokens"], case["heads"], case["dim"]), generator=gen, device=dev) * 1.5
    state["q"] = q.to(DTYPES[case["dtype"]])
    return state


def prepare(case, seed):
    """Inputs of one pass, on the GPU, from the seed."""
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    make = dict(sample=_prepare_sample, plan=_prepare_plan, append=_prepare_append, attend=_prepare_attend)[case["op"]]
    state = make(case, gen, dev)
    if own:
        state.update(_own_handles(state))
    return state


# ---------------------------------------------------------------- this repository's operators
def _package():
    path = str(Path(__file__).resolve().parents[1] / "bitmask-speculation_b200")
    if path not in sys.path:
        sys.path.insert(0, path)


def _own_handles(state):
    _package()
    if state["case"]["op"] == "sample":
        from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
        return dict(call=batched_filtered_sample)
    from bitmask_speculation_b200 import paged
    if state["case"]["op"] == "plan":
        return dict(call=paged.plan_pages)
    cache = paged.PagedCache(state["k"], state["v"])
    return dict(call=paged.rotary_append if state["case"]["op"] == "append" else paged.chunk_attention, cache=cache)


def _own(state):
    case, call = state["case"], state["call"]
    if case["op"] == "sample":
        got = call(state["logits"], state["masks"], uniforms=state["uniforms"], **state["params"])
        return dict(tokens=got.token_ids, kept=got.kept_counts, status=got.status)
    if case["op"] == "plan":
        got = call(state["past"], state["new"], state["held"], state["table"], state["free"], state["count"],
                   page_size=case["page"], tokens=state["tokens"])
        return dict(query_start=got.query_start, seq_lens=got.seq_lens, positions=got.positions, slots=got.slots, held=got.held,
                    count=got.free_count, status=got.status, table=state["table"], free=state["free"])
    if case["op"] == "append":
        q = call(state["q"], state["key"], state["value"], state["cos"], state["sin"], state["positions"], state["slots"], state["cache"])
        return dict(q=q, k=state["k"], v=state["v"])
    got = call(state["q"], state["cache"], state["table"], state["seq_lens"], state["query_start"], window=case["window"], sinks=case["sinks"])
    return dict(out=got.out, lse=got.lse, status=got.status)


# ---------------------------------------------------------------- plain forms
def _rows_of(param, r0, n, device, dtype=torch.float64):
    """A parameter's values for rows [r0, r0 + n) as an [n, 1] column."""
    if isinstance(param, torch.Tensor):
        return param[r0:r0 + n].to(dtype)[:, None]
    return torch.full((n, 1), param, dtype=dtype, device=device)


def _plain_sample(state):
    logits, masks, uniforms, params = state["logits"], state["masks"], state["uniforms"], state["params"]
    rows, vocab = logits.shape
    dev = logits.device
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    kept = torch.empty(rows, dtype=torch.int64, device=dev)
    status = torch.empty(rows, dtype=torch.int32, device=dev)
    shifts = torch.arange(32, device=dev, dtype=torch.int32)
    rank = torch.arange(vocab, device=dev)
    step = max(1, BLOCK // 2 // vocab)
    for r0 in range(0, rows, step):
        n = min(step, rows - r0)
        temp, k, p, floor = (_rows_of(params[name], r0, n, dev) for name in ("temperature", "top_k", "top_p", "min_p"))
        valid = ((masks[r0:r0 + n, :, None] >> shifts) & 1).view(n, -1)[:, :vocab] != 0
        x = logits[r0:r0 + n].float()
        nan = torch.isnan(x).any(1)
        x = torch.where(valid, x, -math.inf)
        empty = ~valid.any(1)
        finite = (x > -math.inf).sum(1, keepdim=True)
        order_x, order = x.sort(dim=1, descending=True, stable=True)  # equal scores stay in the order of their tokens
        top = order_x[:, :1].double()
        scale = torch.where(temp > 0, temp, 1.0)
        weight = ((order_x.double() - top) / scale).exp()
        limit = torch.where(k > 0, torch.minimum(k, finite), finite)
        weight = torch.where(rank < limit, weight, 0.0)
        total = weight.cumsum(1)
        before = torch.nn.functional.pad(total[:, :-1], (1, 0))
        keep = (rank < limit) & ((p >= 1) | (before < p * total[:, -1:])) & (weight >= floor)
        count = keep.sum(1)
        weight = torch.where(keep, weight, 0.0)
        mass = torch.zeros_like(weight).scatter_(1, order, weight).cumsum(1)
        above = mass > uniforms[r0:r0 + n, None] * mass[:, -1:]
        last = (mass >= mass[:, -1:]).int().argmax(1)
        token = torch.where(above.any(1), above.int().argmax(1), last)
        greedy = temp[:, 0] == 0
        token = torch.where(greedy, order[:, 0], token)
        count = torch.where(greedy, 1, count)
        code = torch.zeros(n, dtype=torch.int32, device=dev)
        code = torch.where(~greedy & (finite[:, 0] == 0), 4, code)
        code = torch.where(empty, 1, code)
        code = torch.where(~greedy & (top[:, 0] == math.inf), 5, code)
        code = torch.where(nan, 2, code)
        tokens[r0:r0 + n] = torch.where(code == 0, token, -1)
        kept[r0:r0 + n] = torch.where(code == 0, count, 0)
        status[r0:r0 + n] = code
    return dict(tokens=tokens, kept=kept, status=status)


def _plain_plan(state):
    case, table, free = state["case"], state["table"], state["free"]
    page, tokens = case["page"], state["tokens"]
    dev = table.device
    seqs, width = table.shape
    pages = free.numel()
    past, new, held = (state[name].long() for name in ("past", "new", "held"))
    count = state["count"].long().clamp(0, pages)
    rows = new.clamp(min=0)
    start = torch.nn.functional.pad(rows.cumsum(0), (1, 0))
    good = (past >= 0) & (new >= 0) & (held >= 0) & (held <= width) & (past <= held * page) & (past + new <= width * page) & (start[1:] <= tokens)
    need = torch.where(good, (past + new + page - 1) // page, held)
    grab, drop = (need - held).clamp(min=0), (held - need).clamp(min=0)
    dropped = torch.nn.functional.pad(drop.cumsum(0), (1, 0))
    grabbed = grab.cumsum(0)
    level = count + dropped[-1]  # pages that can be handed out: the free ones, then those given back now
    enough = (grab == 0) | (grabbed <= level)
    good, grab = good & enough, torch.where(enough, grab, 0)
    cell = torch.arange(width, device=dev)[None, :]
    # The stack: the free pages, then every given-back page in the order of sequences and entries.
    stack = torch.cat([free.long(), torch.zeros(seqs * width, dtype=torch.int64, device=dev)])
    back = (cell >= need[:, None]) & (cell < held[:, None]) & (drop[:, None] > 0)
    at = (count + dropped[:-1])[:, None] + cell - need[:, None]
    stack[at[back]] = table.long()[back]
    take = (cell >= held[:, None]) & (cell < (held + grab)[:, None])
    at = (level - 1 - (grabbed - grab))[:, None] - (cell - held[:, None])
    table[take] = stack[at[take]].to(torch.int32)
    left = (level - grab.sum()).clamp(max=pages)
    entry = torch.arange(pages, device=dev)
    kept_back = (entry >= count) & (entry < left)
    free[kept_back] = stack[:pages][kept_back].to(torch.int32)
    index = torch.arange(tokens, device=dev)
    seq = torch.searchsorted(start[1:].contiguous(), index, right=True).clamp(max=seqs - 1)
    live = (index < start[-1]) & good[seq]
    position = torch.where(live, past[seq] + index - start[seq], -1)
    slot_page = table[seq, (position.clamp(min=0) // page).clamp(max=width - 1)].long()
    slots = torch.where(live & (slot_page >= 0) & (slot_page < pages), slot_page * page + position % page, -1)
    code = torch.where(good, 0, torch.where(enough, 6, 9)).to(torch.int32)
    return dict(query_start=start.clamp(max=tokens).to(torch.int32), seq_lens=torch.where(good, past + new, 0).to(torch.int32),
                positions=position.to(torch.int32), slots=slots, held=torch.where(good, need, held).to(torch.int32),
                count=left.to(torch.int32), status=code, table=table, free=free)


def _turn(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _plain_append(state, wide=torch.float32):
    k, v, slots = state["k"], state["v"], state["slots"]
    at = state["positions"].long()
    cos, sin = state["cos"][at][:, None].to(wide), state["sin"][at][:, None].to(wide)
    out_type = k.dtype if wide is torch.float32 else wide
    q = _turn(state["q"].to(wide), cos, sin).to(out_type)
    flat_k, flat_v = (c.view(-1, *c.shape[2:]) for c in (k, v))
    flat_k[slots] = _turn(state["key"].to(wide), cos, sin).to(out_type)
    flat_v[slots] = state["value"].to(out_type)
    return dict(q=q, k=k, v=v)


def _plain_attend(state, wide=torch.float32):
    case, q = state["case"], state["q"]
    heads, kv_heads, dim, window, sinks = case["heads"], case["kv_heads"], case["dim"], case["window"], case["sinks"]
    dev = q.device
    out = torch.zeros(q.shape, dtype=q.dtype if wide is torch.float32 else wide, device=dev)
    lse = torch.full(q.shape[:2], -math.inf, dtype=wide, device=dev)
    page, row = case["page"], 0
    for s, (n, past) in enumerate(zip(state["new"], state["past"])):
        length = n + past
        table = state["table"][s, :-(-length // page)].long()
        k, v = (state[name][table].view(-1, kv_heads, dim)[:length].to(wide).transpose(0, 1) for name in ("k", "v"))
        key = torch.arange(length, device=dev)
        step = max(1, BLOCK // (heads * length)) if length else 1
        for r0 in range(0, n, step):
            m = min(step, n - r0)
            position = past + r0 + torch.arange(m, device=dev)[:, None]
            seen = key <= position
            if window:
                seen = seen & ((position - key < window) | (key < sinks))
            part = q[row + r0:row + r0 + m].to(wide).view(m, kv_heads, heads // kv_heads, dim).permute(1, 2, 0, 3)
            score = torch.matmul(part.reshape(kv_heads, -1, dim), k.transpose(1, 2)) / math.sqrt(dim)
            score = torch.where(seen, score.view(kv_heads, heads // kv_heads, m, length), -math.inf)
            top = score.amax(-1, keepdim=True)
            weight = (score - top).exp()
            total = weight.sum(-1, keepdim=True)
            got = torch.matmul(weight.view(kv_heads, -1, length), v).view(kv_heads, -1, m, dim) / total
            out[row + r0:row + r0 + m] = got.permute(2, 0, 1, 3).reshape(m, heads, dim).to(out.dtype)
            lse[row + r0:row + r0 + m] = (top + total.log())[..., 0].permute(2, 0, 1).reshape(m, heads)
        row += n
    return dict(out=out, lse=lse, status=torch.zeros(case["seqs"], dtype=torch.int32, device=dev))


def run(state):
    """One pass through the case's operator."""
    if own:
        return _own(state)
    return dict(sample=_plain_sample, plan=_plain_plan, append=_plain_append, attend=_plain_attend)[state["case"]["op"]](state)


# ---------------------------------------------------------------- work
def work(case):
    """Bytes that have to move and operations that have to be done in one pass."""
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": rows * (vocab * size + (vocab + 31) // 32 * 4 + 8 + 20), "flops": 2 * rows * vocab}
    new, past = _lengths(case)
    if case["op"] == "plan":
        page = case["page"]
        grown = sum(max(0, -(-(p + n) // page) - -(-p // page)) for p, n in zip(past, new))
        return {"bytes": case["seqs"] * 4 * (3 + 4) + 8 * grown + sum(new) * 12, "flops": sum(new)}
    size = 4 if case["dtype"] == "float32" else 2
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        values = sum(new) * (heads + 2 * kv_heads) * dim
        return {"bytes": 2 * values * size + sum(new) * 12 + len({p + i for p, n in zip(past, new) for i in range(n)}) * dim * 4,
                "flops": 3 * sum(new) * (heads + kv_heads) * dim}
    keys = pairs = 0
    for n, p in zip(new, past):
        if n == 0:
            continue
        w, sinks = case["window"] or n + p, case["sinks"]
        first = max(0, p + 1 - w)
        keys += n + p - first + min(sinks, first)
        for i in range(n):
            low = max(0, p + i + 1 - w)
            pairs += p + i + 1 - low + min(sinks, low)
    rows = sum(new) * heads
    return {"bytes": 2 * rows * dim * size + rows * 4 + 2 * keys * kv_heads * dim * size + case["seqs"] * 12, "flops": 4 * pairs * heads * dim}


# ---------------------------------------------------------------- definitions in 64 bits
def _exact_sample_row(x, valid, temperature, k, p, floor, u):
    """(token, kept, status) of one row, from the definition."""
    if np.isnan(x).any():
        return -1, 0, 2
    ids = np.flatnonzero(valid)
    if temperature > 0 and ids.size and x[ids].max() == np.inf:
        return -1, 0, 5
    if not ids.size:
        return -1, 0, 1
    if temperature == 0:
        return int(ids[np.argmax(x[ids])]), 1, 0
    ids = ids[x[ids] > -np.inf]
    if not ids.size:
        return -1, 0, 4
    ids = ids[np.lexsort((ids, -x[ids]))]
    if k > 0:
        ids = ids[:k]
    w = np.exp((x[ids] - x[ids[0]]) / temperature)
    n = ids.size
    if p < 1:
        c = np.cumsum(w)
        n = min(n, int(np.searchsorted(c, p * c[-1], side="left")) + 1)
    n = min(n, int((w >= floor).sum()))
    ids, w = ids[:n], w[:n]
    by_id = np.argsort(ids)
    c = np.cumsum(w[by_id])
    at = min(int(np.searchsorted(c, u * c[-1], side="right")), int(np.searchsorted(c, c[-1], side="left")))
    return int(ids[by_id][at]), n, 0


def _exact_sample(state):
    case = state["case"]
    if case["rows"] * case["vocab"] > 50_000_000:
        return None
    masks = state["masks"].cpu().numpy()
    valid = np.unpackbits(np.ascontiguousarray(masks).view(np.uint8), axis=1, bitorder="little")[:, :case["vocab"]].astype(bool)
    u = state["uniforms"].cpu().numpy()
    params = {name: np.broadcast_to(value.double().cpu().numpy() if isinstance(value, torch.Tensor) else value, (case["rows"],))
              for name, value in state["params"].items()}
    rows = [_exact_sample_row(state["logits"][r].double().cpu().numpy(), valid[r], params["temperature"][r], int(params["top_k"][r]),
                              params["top_p"][r], params["min_p"][r], u[r]) for r in range(case["rows"])]
    return dict(tokens=np.array([r[0] for r in rows], dtype=np.int64), kept=np.array([r[1] for r in rows], dtype=np.int64),
                status=np.array([r[2] for r in rows], dtype=np.int32))


def _exact_attend(state):
    """Scores, weights and sums in 64 bits, one head and one block of rows at a time."""
    case, q = state["case"], state["q"]
    if work(case)["flops"] > 4e12:
        return None
    group, dim, page = case["heads"] // case["kv_heads"], case["dim"], case["page"]
    dev = q.device
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=dev)
    row = 0
    for s, (n, past) in enumerate(zip(state["new"], state["past"])):
        at = torch.arange(n + past, device=dev)
        pages = state["table"][s].long()[at // page]
        for h in range(case["kv_heads"] if n else 0):
            k, v = state["k"][pages, at % page, h].double(), state["v"][pages, at % page, h].double()
            for r0 in range(0, n, 1024):
                r1 = min(n, r0 + 1024)
                age = torch.arange(past + r0, past + r1, device=dev)[:, None] - at[None, :]
                hidden = age < 0
                if case["window"]:
                    hidden |= (age >= case["window"]) & (at[None, :] >= case["sinks"])
                for j in range(h * group, (h + 1) * group):
                    score = (q[row + r0:row + r1, j].double() @ k.T) * dim ** -0.5
                    score.masked_fill_(hidden, -math.inf)
                    norm = torch.logsumexp(score, 1, keepdim=True)
                    out[row + r0:row + r1, j] = (score - norm).exp_() @ v
                    lse[row + r0:row + r1, j] = norm[:, 0]
        row += n
    return dict(out=out, lse=lse, status=None)


def _exact_append(state):
    at = state["positions"].long().cpu()
    cos, sin = state["cos"].cpu().double()[at].numpy()[:, None], state["sin"].cpu().double()[at].numpy()[:, None]
    slots = state["slots"].cpu().numpy()

    def turned(x):
        x = x.cpu().double().numpy()
        a, b = np.split(x, 2, axis=-1)
        return np.concatenate((a * cos - b * sin, b * cos + a * sin), -1)

    k, v = (state[name].cpu().double().numpy() for name in ("k", "v"))
    k.reshape(-1, *k.shape[2:])[slots] = turned(state["key"])
    v.reshape(-1, *v.shape[2:])[slots] = state["value"].cpu().double().numpy()
    return dict(q=turned(state["q"]), k=k, v=v)


def exact(case, seed):
    """What ``run`` returns, from each operator's definition in 64 bits; None where that takes long or no value is computed."""
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "plan":
        return None
    return dict(sample=_exact_sample, append=_exact_append, attend=_exact_attend)[case["op"]](state)
