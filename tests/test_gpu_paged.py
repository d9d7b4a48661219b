"""Paged cache operators against plain float64 forms: page planning, rotary append, chunk attention, and a run of
all of them together."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}  # torch.finfo(t).eps


# ---------------------------------------------------------------- page plan
def plan_definition(past, new, held, table, free, count, page, tokens):
    """The plan's sequential definition on Python lists."""
    table, free = [list(r) for r in table], list(free)
    width, pages = len(table[0]), len(free)
    count = max(0, min(count, pages))
    starts, need, good = [0], [], []
    for s, (p, n, h) in enumerate(zip(past, new, held)):
        starts.append(starts[-1] + max(n, 0))
        ok = p >= 0 and n >= 0 and 0 <= h <= width and p <= h * page and p + n <= width * page and starts[-1] <= tokens
        good.append(ok)
        need.append(-(-(p + n) // page) if ok else h)
    stack = free[:count]
    for s in range(len(past)):
        if good[s]:
            stack += table[s][need[s]:held[s]]
    asked, status, level = 0, [], len(stack)
    for s in range(len(past)):
        status.append(0 if good[s] else 6)
        if need[s] > held[s]:
            asked += need[s] - held[s]
            if asked <= level:
                for i in range(held[s], need[s]):
                    table[s][i] = stack.pop()
            else:
                status[s] = 9
    positions, slots = [-1] * tokens, [-1] * tokens
    for s in range(len(past)):
        if status[s]:
            continue
        for i in range(new[s]):
            pos = past[s] + i
            pg = table[s][pos // page]
            positions[starts[s] + i] = pos
            slots[starts[s] + i] = pg * page + pos % page if 0 <= pg < pages else -1
    stack = stack[:pages]
    free[count:len(stack)] = stack[count:]
    return dict(query_start=[min(a, tokens) for a in starts], seq_lens=[p + n if not st else 0 for p, n, st in zip(past, new, status)],
                positions=positions, slots=slots, held=[h if st else m for h, m, st in zip(held, need, status)], free_count=[len(stack)],
                status=status), table, free


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check_plan(past, new, held, table, free, count, page, tokens):
    from bitmask_speculation_b200.paged import plan_pages
    want, want_table, want_free = plan_definition(past, new, held, table, free, count, page, tokens)
    t, f = i32(table), i32(free)
    for _ in range(2):  # the same call again gives the same result
        got = plan_pages(i32(past), i32(new), i32(held), t, f, i32([count]), page_size=page, tokens=tokens)
        for name, value in want.items():
            assert getattr(got, name).tolist() == value, name
        assert t.tolist() == want_table
        assert f.tolist() == want_free
    return got


def random_plan(rng, seqs, page, width, spare, tokens_slack=0):
    past = [int(rng.integers(0, width * page // 2 + 1)) for _ in range(seqs)]
    new = [int(rng.integers(0, width * page // 2 + 1)) if rng.random() < 0.8 else 0 for _ in range(seqs)]
    held = [min(width, -(-p // page) + int(rng.choice([0, 0, 1, 3]))) for p in past]
    pages = sum(held) + spare
    order = [int(v) for v in rng.permutation(pages)]
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [0] * (width - h))
        at += h
    free = order[at:] + [0] * at
    return past, new, held, table, free, spare, page, sum(new) + tokens_slack


@pytest.mark.parametrize("seqs,page,width", [(1, 1, 1), (1, 16, 4), (7, 5, 9), (33, 16, 12), (600, 8, 6), (1500, 4, 5)])
def test_plans(cuda_module, seqs, page, width):
    rng = np.random.default_rng(seqs)
    for spare in (0, 1, seqs, seqs * width):  # from an exhausted pool to an ample one
        check_plan(*random_plan(rng, seqs, page, width, spare, tokens_slack=int(rng.integers(0, 5))))


def test_plan_of_nothing_and_finished_requests(cuda_module):
    check_plan([0, 0, 0], [0, 0, 0], [0, 2, 3], [[9, 9, 9], [4, 1, 9], [0, 2, 3]], [7, 5, 6, 0, 0, 0, 0, 0, 0, 0], 3, 4, 0)
    # What one request gives back another takes in the same call.
    got = check_plan([0, 1], [0, 11], [3, 1], [[4, 1, 2], [0, 7, 7]], [3, 0, 0, 0, 0], 1, 4, 11)
    assert got.check() is got and got.free_count.tolist() == [2]


def test_plan_failures(cuda_module):
    table = [[0, 1], [2, 3], [4, 5], [6, 7], [8, 9]]
    free = list(range(10)) + [0] * 10
    args = dict(held=[2, 2, 2, 2, 2], table=table, free=free, count=0, page=4)
    for past, new in (([-1, 0, 0, 0, 0], [1] * 5), ([0] * 5, [-2, 1, 1, 1, 1]), ([9, 1, 1, 1, 1], [0] * 5), ([1] * 5, [1, 2 ** 31 - 1, 1, 1, 1]),
                      ([5, 5, 5, 5, 5], [3, 4, 3, 3, 3])):
        check_plan(past, new, args["held"], table, free, 0, 4, 20)
    check_plan([1] * 5, [3, 3, 3, 3, 3], args["held"], table, free, 0, 4, 10)  # rows behind the capacity
    check_plan([1] * 5, [1] * 5, [2, 3, -1, 2, 2], table, free, 0, 4, 10)
    check_plan([4, 4, 4, 4, 4], [1] * 5, [1, 1, 1, 1, 1], [[0, 1], [2, 3], [4, -5], [6, 7], [8, 99]], free, 3, 4, 5)  # pages outside the pool: no slot
    for count in (-3, 25):
        check_plan([1] * 5, [5] * 5, [1] * 5, table, free, count, 4, 25)
    got = check_plan([0, 0], [4, 5], [0, 0], [[0, 0], [0, 0]], [1, 0, 2], 2, 4, 9)
    with pytest.raises(ValueError, match=r"\(1, 9\)"):
        got.check()


def test_plan_refusals(cuda_module):
    from bitmask_speculation_b200.paged import plan_pages
    one, table, free = i32([0]), i32([[0, 0]]), i32([0, 1, 2])
    ok = dict(page_size=4, tokens=1)
    for args, kw, error in (((one.long(), one, one, table, free, one), ok, TypeError), ((one, i32([0, 1]), one, table, free, one), ok, ValueError),
                            ((one, one, one, table[0], free, one), ok, ValueError), ((one, one, one, table, free, i32([1, 1])), ok, ValueError),
                            ((one, one, one, table.cpu(), free, one), ok, ValueError), ((one, one, one, table, free, one), dict(page_size=0, tokens=1), ValueError),
                            ((one, one, one, table, free, one), dict(page_size=4, tokens=-1), ValueError),
                            ((one, one, one, table, free, one), dict(page_size=4.0, tokens=1), TypeError),
                            ((one, one, one, table[:, :0], free, one), ok, ValueError)):
        with pytest.raises(error):
            plan_pages(*args, **kw)
    big = torch.zeros(8193, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="sequences"):
        plan_pages(big, big, big, big[:, None], free, one, **ok)


# ---------------------------------------------------------------- rotary append
def rotated(x, cos, sin):
    a, b = x.double().chunk(2, -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat((a * c - b * s, a * s + b * c), -1)


def rope_tables(limit, dim):
    inv = 1.0 / (1e6 ** (torch.arange(0, dim, 2, dtype=torch.float64) / dim))
    angle = torch.arange(limit, dtype=torch.float64)[:, None] * inv
    return angle.cos().float().cuda(), angle.sin().float().cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,heads,kv_heads,dim,page", [(1, 4, 1, 64, 16), (9, 3, 3, 128, 5), (70, 8, 2, 80, 1), (33, 5, 5, 6, 7), (500, 16, 4, 64, 32)])
@pytest.mark.parametrize("layout", ["fused", "plain", "odd"])
def test_append(cuda_module, dtype, n, heads, kv_heads, dim, page, layout):
    from bitmask_speculation_b200.paged import PagedCache, rotary_append
    gen = torch.Generator(device="cuda").manual_seed(n * dim)
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda").to(dtype)  # noqa: E731
    pages = n // page + 3
    if layout == "fused":
        fused = rand(n, heads + 2 * kv_heads, dim)
        q, k, v = fused[:, :heads], fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:]
    elif layout == "plain":
        q, k, v = rand(n, heads, dim), rand(n, kv_heads, dim), rand(n, kv_heads, dim)
    else:  # bases off every vector boundary, heads outside tokens
        q, k, v = (rand(h, n, dim + 1)[:, :, 1:].transpose(0, 1) for h in (heads, kv_heads, kv_heads))
    if layout == "odd":
        kc, vc = (rand(pages, kv_heads, page, dim).transpose(1, 2) for _ in range(2))
    else:
        kc, vc = rand(pages, page, kv_heads, dim), rand(pages, page, kv_heads, dim)
    cos, sin = rope_tables(1000, dim)
    positions = torch.randint(1000, (n,), generator=gen, device="cuda", dtype=torch.int32)
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:n]
    skip = torch.arange(n, device="cuda") % 5 == 3
    slots = torch.where(skip, -1, slots)
    gone = torch.arange(n, device="cuda") % 7 == 6
    positions[gone] = -1
    out = torch.full((n, heads, dim), 7.0, dtype=dtype, device="cuda")
    want_k, want_v = kc.clone(), vc.clone()
    cache = PagedCache(kc, vc)
    status = torch.full((n,), 99, dtype=torch.int32, device="cuda")
    assert rotary_append(q, k, v, cos, sin, positions, slots, cache, out=out, status=status) is out
    at = positions.long().clamp(min=0)
    live = (slots >= 0) & ~gone
    # One rounding to the type, and float32 products and sum of two terms: each off by 2^-24 of the terms.
    for got, x in ((out, q), (kc[torch.where(live, slots, 0) // page, torch.where(live, slots, 0) % page], k)):
        want = rotated(x, cos[at], sin[at])
        bound = EPS[dtype] / 2 * want.abs() + 4 * 2.0 ** -24 * (x.double().abs().amax(-1, keepdim=True) * 2) + 2.0 ** -26
        rows = ~gone if got is out else live
        assert bool(((got.double() - want).abs() <= bound)[rows].all())
    assert bool((out[gone] == 7).all())
    s = slots[live]
    want_v[s // page, s % page] = v[live]
    assert torch.equal(vc, want_v)
    want_k[s // page, s % page] = kc[s // page, s % page]
    assert torch.equal(kc, want_k)  # no other slot was written
    assert status.tolist() == [0] * n


def test_append_status_and_refusals(cuda_module):
    from bitmask_speculation_b200.paged import PagedCache, rotary_append
    cache = PagedCache.allocate(4, 8, 2, 64)
    x = torch.ones((5, 2, 64), dtype=torch.bfloat16, device="cuda")
    cos, sin = rope_tables(10, 64)
    positions = i32([0, 9, 10, 5, 2 ** 31 - 1])
    slots = torch.tensor([31, 32, 0, 2 ** 40, -7], device="cuda")
    status = torch.empty(5, dtype=torch.int32, device="cuda")
    rotary_append(x, x, x, cos, sin, positions, slots, cache, status=status)
    assert status.tolist() == [0, 11, 12, 11, 12]
    assert int((cache.v != 0).sum()) == 128 and bool((cache.v[3, 7] == 1).all())
    call = lambda **kw: rotary_append(**{**dict(q=x, k=x, v=x, cos=cos, sin=sin, positions=positions, slots=slots, cache=cache), **kw})  # noqa: E731
    for kw, error in ((dict(q=x.half()), TypeError), (dict(k=x[:4]), ValueError), (dict(k=x[:, :1]), ValueError), (dict(v=x.float()), TypeError),
                      (dict(cos=cos[:, :3]), ValueError), (dict(cos=cos.double()), TypeError), (dict(slots=slots.int()), TypeError),
                      (dict(positions=positions[:3]), ValueError), (dict(out=x[:, :1]), ValueError), (dict(q=x.transpose(1, 2)[:, :2, :]), ValueError),
                      (dict(q=x.expand(5, 2, 64)[..., :32]), ValueError), (dict(positions=positions.cpu()), ValueError)):
        with pytest.raises(error):
            call(**kw)
    rotary_append(x[:0], x[:0], x[:0], cos, sin, positions[:0], slots[:0], cache)
    with pytest.raises(ValueError):
        PagedCache(cache.k, cache.v[:3])
    with pytest.raises(TypeError):
        PagedCache(cache.k.double(), cache.v.double())
    with pytest.raises(ValueError):
        PagedCache(cache.k.transpose(2, 3), cache.v.transpose(2, 3))


# ---------------------------------------------------------------- chunk attention
def make_case(lens, heads, kv_heads, dim, page, dtype, seed=0, poison=True, sharp=1.0):
    """Queries, a cache whose unused slots and pages hold NaN and infinities, tables in no order."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-(n + p) // page) for n, p in lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=gen, device="cuda").tolist()
    width = max(max(need), 1) + 1
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    k = torch.randn((pages, page, kv_heads, dim), generator=gen, device="cuda").to(dtype)
    v = torch.randn((pages, page, kv_heads, dim), generator=gen, device="cuda").to(dtype)
    used = torch.zeros((pages, page), dtype=torch.bool)
    at = 0
    for s, m in enumerate(need):
        mine = order[at:at + m]
        at += m
        table[s, :m] = torch.tensor(mine, dtype=torch.int32)
        for i in range(sum(lens[s])):
            used[mine[i // page], i % page] = True
    if poison:
        k[~used.cuda()] = math.nan
        v[~used.cuda()] = math.inf
    q = (torch.randn((sum(n for n, _ in lens), heads, dim), generator=gen, device="cuda") * sharp).to(dtype)
    starts = i32([0] + list(np.cumsum([n for n, _ in lens])))
    return q, k, v, table.cuda(), i32([n + p for n, p in lens]), starts


def definition(q, k, v, table, lens, window, sinks, scale):
    """(out, lse, sum of p |v|, largest scale sum |q k|) in float64."""
    heads, dim = q.shape[1:]
    page, kv_heads = k.shape[1], k.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    weight, size = torch.zeros_like(out), torch.zeros_like(lse)
    row = 0
    for s, (n, past) in enumerate(lens):
        if n == 0:
            continue
        at = torch.arange(n + past, device="cuda")
        pg = table[s].long()[at // page].clamp(min=0)
        ks, vs = k[pg, at % page].double(), v[pg, at % page].double()
        age = (past + torch.arange(n, device="cuda"))[:, None] - at
        seen = age >= 0
        if window:
            seen &= (age < window) | (at < sinks)
        for h in range(heads):
            j = h // (heads // kv_heads)
            kk, vv = torch.nan_to_num(ks[:, j], 0, 0, 0), torch.nan_to_num(vs[:, j], 0, 0, 0)
            qq = q[row:row + n, h].double()
            score = (qq @ kk.T * scale).masked_fill(~seen, -math.inf)
            norm = torch.logsumexp(score, 1, keepdim=True)
            p = (score - norm).exp()
            out[row:row + n, h], lse[row:row + n, h] = p @ vv, norm[:, 0]
            weight[row:row + n, h] = p @ vv.abs()
            size[row:row + n, h] = (qq.abs() @ kk.abs().T * abs(scale)).masked_fill(~seen, 0).amax(1)
        row += n
    return out, lse, weight, size


def assert_close(got, want, dtype, dim):
    out, lse, weight, size = want
    # Scores: float32 sums of dim products, the scale and the base change, off by (dim + 4) 2^-24 of the terms;
    # exponentials and their sums 2^-20; each weight rounded once to the inputs' type, the result once.
    score = (dim + 4) * 2.0 ** -24 * size + 2.0 ** -20
    half = EPS[dtype] / 2
    low = 0 if dtype is torch.float32 else half
    bound = (low + 2 * score[..., None]) * weight * (1 + half) + half * out.abs() + (2.0 ** -24 if dtype is torch.float16 else 2.0 ** -126)
    assert bool(((got.out.double() - out).abs() <= bound).all()), float(((got.out.double() - out).abs() / bound).max())
    fine = torch.isfinite(lse)
    assert torch.equal(fine, torch.isfinite(got.lse))
    assert bool(((got.lse.double() - lse).abs() <= score + 2.0 ** -22 * (1 + lse.abs()))[fine].all())


def check_attention(lens, heads, kv_heads, dim, page, dtype, window=0, sinks=0, scale=None, **kw):
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    q, k, v, table, seq_lens, starts = make_case(lens, heads, kv_heads, dim, page, dtype, **kw)
    got = chunk_attention(q, PagedCache(k, v), table, seq_lens, starts, window=window, sinks=sinks, scale=scale)
    assert got.status.tolist() == [0] * len(lens)
    assert_close(got, definition(q, k, v, table, lens, window, sinks, dim ** -0.5 if scale is None else scale), dtype, dim)


LENS = {
    "one": [(1, 0)],
    "decode": [(1, 0), (1, 1), (1, 127), (1, 128), (1, 129), (1, 700), (1, 63)],
    "round": [(9, 300), (9, 0), (9, 119), (1, 200), (0, 50), (9, 1000)],
    "chunks": [(300, 0), (0, 0), (130, 257), (1, 5), (64, 64), (33, 900)],
    "empty": [(0, 0), (0, 10), (2, 3), (0, 0)],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 1, 64, 16), (8, 8, 128, 32), (6, 2, 64, 64), (28, 4, 128, 128), (5, 1, 80, 5), (2, 1, 256, 16), (3, 3, 40, 1),
                                                     (32, 1, 64, 16)])
@pytest.mark.parametrize("lens", list(LENS))
def test_attention(cuda_module, dtype, heads, kv_heads, dim, page, lens):
    check_attention(LENS[lens], heads, kv_heads, dim, page, dtype)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (7, 0), (100, 4), (128, 130), (5000, 2), (64, 1000)])
def test_window_and_sinks(cuda_module, dtype, dim, window, sinks):
    for lens in ("decode", "round", "chunks"):
        check_attention(LENS[lens], 8, 2, dim, 16, dtype, window, sinks)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_scales(cuda_module, scale):
    check_attention(LENS["round"], 4, 2, 64, 16, torch.float16, scale=scale)


def test_sharp_scores_over_long_caches(cuda_module):
    """Running maxima that jump late, weights that underflow."""
    for dtype in (torch.bfloat16, torch.float16):
        check_attention([(1, 9000), (9, 5000), (200, 3000)], 8, 2, 128, 32, dtype, sharp=6.0, scale=0.5)


def test_long_single_sequence(cuda_module):
    check_attention([(1, 40000)], 4, 1, 64, 16, torch.bfloat16)
    check_attention([(1, 40000)], 4, 1, 128, 128, torch.float16, window=30000, sinks=5)


def test_hidden_keys_never_reach_a_row(cuda_module):
    """NaN and infinities in keys and values that some rows see and others do not: the rows that do not
    see them are those of the clean cache, bit for bit in their bound."""
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    for dtype, dim in ((torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64)):
        lens = [(40, 100), (9, 10), (300, 7)]
        q, k, v, table, seq_lens, starts = make_case(lens, 8, 2, dim, 16, dtype)
        want = definition(q, k, v, table, lens, 0, 0, dim ** -0.5)
        clean = chunk_attention(q, PagedCache(k, v), table, seq_lens, starts)
        row = 0
        hidden = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
        for s, (n, past) in enumerate(lens):
            bad = past + n // 2  # the middle new token: later rows see it, earlier ones do not
            pg = int(table[s, bad // 16])
            k[pg, bad % 16] = math.nan
            v[pg, bad % 16, :, ::3] = math.inf
            v[pg, bad % 16, :, 1::3] = math.nan
            hidden[row + n // 2:row + n] = False
            row += n
        got = chunk_attention(q, PagedCache(k, v), table, seq_lens, starts)
        out, lse, weight, size = (t[hidden] for t in want)
        clean = type(got)(clean.out[hidden], clean.lse[hidden], clean.status)
        assert_close(type(got)(got.out[hidden], got.lse[hidden], got.status), (out, lse, weight, size), dtype, dim)
        assert_close(clean, (out, lse, weight, size), dtype, dim)
        assert bool(torch.isnan(got.out[~hidden]).all())


def test_hidden_behind_a_window(cuda_module):
    """Pages that slid out of every row's window may hold anything, or lie outside the cache."""
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    for dtype in (torch.bfloat16, torch.float32):
        lens, window, sinks = [(5, 600), (1, 900)], 50, 2
        q, k, v, table, seq_lens, starts = make_case(lens, 4, 1, 64, 16, dtype)
        want = definition(q, k, v, table, lens, window, sinks, 0.125)
        for s, (n, past) in enumerate(lens):
            first = past + 1 - window  # the lowest key that any row sees beside the sinks
            for j in range(sinks, first):
                pg = int(table[s, j // 16])
                k[pg, j % 16], v[pg, j % 16] = math.inf, math.nan
            table[s, 1:first // 16] = 10 ** 6
        got = chunk_attention(q, PagedCache(k, v), table, seq_lens, starts, window=window, sinks=sinks)
        assert got.status.tolist() == [0, 0]
        assert_close(got, want, dtype, 64)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 40)])
def test_failed_sequences(cuda_module, dtype, dim):
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    lens = [(3, 30), (4, 100), (20, 500), (1, 0), (9, 200)]
    q, k, v, table, seq_lens, starts = make_case(lens, 4, 2, dim, 16, dtype)
    want = definition(q, k, v, table, lens, 0, 0, dim ** -0.5)
    table[1, 2], table[4, 0] = k.shape[0], -1
    seq_lens[2] = 19
    out = torch.full(q.shape, 5.0, dtype=dtype, device="cuda")
    got = chunk_attention(q, PagedCache(k, v), table, seq_lens, starts, out=out)
    assert got.out is out and got.status.tolist() == [0, 11, 6, 0, 11]
    rows = torch.tensor([0] * 3 + [1] * 4 + [2] * 20 + [3] + [4] * 9, device="cuda")
    fine = (rows == 0) | (rows == 3)
    assert_close(type(got)(got.out[fine], got.lse[fine], got.status), tuple(t[fine] for t in want), dtype, dim)
    assert bool((got.out[~fine] == 0).all()) and bool((got.lse[~fine] == -math.inf).all())
    with pytest.raises(ValueError, match=r"\(1, 11\)"):
        got.check()
    seq_lens[0] = 10 ** 6
    assert chunk_attention(q, PagedCache(k, v), table, seq_lens, starts).status.tolist() == [6, 11, 6, 0, 11]
    bad_starts = starts.clone()
    bad_starts[5] = 1000
    assert chunk_attention(q, PagedCache(k, v), table, seq_lens, bad_starts).status.tolist()[4] == 6
    bad_starts[0], bad_starts[5] = -4, 36
    assert chunk_attention(q, PagedCache(k, v), table, seq_lens, bad_starts).status.tolist()[0] == 6


def test_rows_behind_the_last_sequence(cuda_module):
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    for dtype in (torch.bfloat16, torch.float32):
        lens = [(5, 40), (2, 0)]
        q, k, v, table, seq_lens, starts = make_case(lens, 4, 2, 64, 16, dtype)
        padded = torch.cat((q, torch.full((30, 4, 64), math.nan, dtype=dtype, device="cuda")))
        out = torch.full(padded.shape, 3.0, dtype=dtype, device="cuda")
        got = chunk_attention(padded, PagedCache(k, v), table, seq_lens, starts, out=out)
        assert bool((out[7:] == 3).all())
        assert torch.equal(out[:7], chunk_attention(q, PagedCache(k, v), table, seq_lens, starts).out) and got.status.tolist() == [0, 0]


def test_strides_and_layouts(cuda_module):
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    for dtype, page in ((torch.bfloat16, 16), (torch.float16, 64), (torch.float32, 16)):
        lens = LENS["chunks"]
        q, k, v, table, seq_lens, starts = make_case(lens, 8, 2, 64, page, dtype, poison=False)
        want = definition(q, k, v, table, lens, 0, 0, 0.125)
        # Heads outside slots; queries inside one projection's output; an interleaved key/value pool; bases off a vector boundary.
        heads_first = PagedCache(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)))
        pool = torch.stack((k, v), 1)
        interleaved = PagedCache(pool[:, 0], pool[:, 1])
        odd = torch.empty(k.numel() + 3, dtype=dtype, device="cuda")
        odd[3:] = k.flatten()
        unaligned = PagedCache(odd[3:].view(k.shape), v)
        fused = torch.cat((q, q, q), 1)[:, 8:16]
        shifted = torch.nn.functional.pad(q, (1, 2))[..., 1:65]
        for cache in (heads_first, interleaved, unaligned):
            for rows in (q, fused, shifted):
                got = chunk_attention(rows, cache, table, seq_lens, starts)
                assert_close(got, want, dtype, 64)


def test_streams_graphs_and_concurrent_calls(cuda_module):
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    sets = [make_case([(9, 500), (1, 3000), (40, 20)], 8, 2, 128, 32, torch.bfloat16, seed=i) for i in range(2)]
    call = lambda c: chunk_attention(c[0], PagedCache(c[1], c[2]), *c[3:])  # noqa: E731
    want = [call(c).out.clone() for c in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(5):
        for c, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(call(c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g.out, want[i % 2])
    graphs, held = [], []
    for c in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(call(c))
        graphs.append(graph)
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for h, w in zip(held, want):
        assert torch.equal(h.out, w)


def test_attention_refusals(cuda_module):
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    q, k, v, table, seq_lens, starts = make_case([(2, 3)], 4, 2, 64, 16, torch.bfloat16)
    cache = PagedCache(k, v)
    call = lambda **kw: chunk_attention(**{**dict(q=q, cache=cache, block_table=table, seq_lens=seq_lens, query_start=starts), **kw})  # noqa: E731
    for kw, error in ((dict(q=q.half()), TypeError), (dict(q=q[:, :3]), ValueError), (dict(q=q[..., :32]), ValueError), (dict(seq_lens=seq_lens.long()), TypeError),
                      (dict(query_start=starts[:1]), ValueError), (dict(block_table=table[:, :0]), ValueError), (dict(window=-1), ValueError), (dict(sinks=-1), ValueError),
                      (dict(window=1.0), TypeError), (dict(scale="1"), TypeError), (dict(scale=math.inf), ValueError), (dict(out=q[:1]), ValueError),
                      (dict(q=q.transpose(0, 2)), ValueError), (dict(seq_lens=seq_lens.cpu()), ValueError)):
        with pytest.raises(error):
            call(**kw)
    wide = torch.zeros((4, 4, 2, 512), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        chunk_attention(torch.zeros((1, 2, 512), dtype=torch.bfloat16, device="cuda"), PagedCache(wide, wide.clone()), table, seq_lens, starts)
    none = chunk_attention(q[:0], cache, table, i32([7]), i32([0, 0]))
    assert none.out.shape == (0, 4, 64) and none.status.tolist() == [0]


# ---------------------------------------------------------------- a run of them together
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rounds_of_plan_append_attend(cuda_module, dtype):
    """Prompts, drafted windows, rollbacks, a finished request whose pages the next one takes: every
    round's attention equals the definition over the tokens that each sequence has kept."""
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention, plan_pages, rotary_append
    heads, kv_heads, dim, page, seqs, width = 4, 2, 64, 16, 3, 12
    gen = torch.Generator(device="cuda").manual_seed(1)
    cache = PagedCache.allocate(20, page, kv_heads, dim, dtype=dtype)
    cache.k.fill_(math.nan)
    cache.v.fill_(math.nan)
    cos, sin = rope_tables(width * page, dim)
    table, held = torch.zeros((seqs, width), dtype=torch.int32, device="cuda"), i32([0] * seqs)
    free, count = torch.arange(20, dtype=torch.int32, device="cuda"), i32([20])
    kept = [[] for _ in range(seqs)]  # each sequence's (key, value) rows
    rounds = [([0, 0, 0], [40, 17, 0]), ([40, 17, 0], [9, 9, 130]), ([43, 26, 130], [9, 9, 1]), ([0, 27, 131], [0, 9, 1]), ([0, 36, 0], [100, 1, 0])]
    for past, new in rounds:
        n = sum(new)
        plan = plan_pages(i32(past), i32(new), held, table, free, count, page_size=page, tokens=n + 2).check()
        held, count = plan.held, plan.free_count
        assert int(held.sum()) + int(count) == 20
        q, k, v = (torch.randn((n + 2, h, dim), generator=gen, device="cuda").to(dtype) for h in (heads, kv_heads, kv_heads))
        turned = rotary_append(q, k, v, cos, sin, plan.positions, plan.slots, cache)
        got = chunk_attention(turned, cache, table, plan.seq_lens, plan.query_start).check()
        row = 0
        for s in range(seqs):
            rows = slice(row, row + new[s])
            row += new[s]
            at = plan.positions[rows].long()
            k_rows, v_rows = (t.reshape(-1, kv_heads, dim)[plan.slots[rows]] for t in (cache.k, cache.v))
            exact = rotated(k[rows], cos[at], sin[at])
            assert bool(((k_rows.double() - exact).abs() <= EPS[dtype] / 2 * exact.abs() + 2.0 ** -20).all()) and torch.equal(v_rows, v[rows])
            kept[s] = kept[s][:past[s]] + list(zip(k_rows, v_rows))
            if not new[s]:
                continue
            ks, vs = (torch.stack([pair[i] for pair in kept[s]])[None] for i in range(2))
            want = definition(turned[rows], ks, vs, i32([[0]]), [(new[s], past[s])], 0, 0, dim ** -0.5)
            assert_close(type(got)(got.out[rows], got.lse[rows], got.status), want, dtype, dim)


def test_broadcast_queries(cuda_module):
    """Queries expanded over heads or tokens (strides of 0)."""
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    lens = [(9, 200), (70, 30), (1, 5)]
    q, k, v, table, seq_lens, starts = make_case(lens, 8, 2, 64, 16, torch.bfloat16)
    for rows in (q[:, :1].expand(-1, 8, -1), q[:1].expand(80, -1, -1)):
        got = chunk_attention(rows, PagedCache(k, v), table, seq_lens, starts)
        assert_close(got, definition(rows.contiguous(), k, v, table, lens, 0, 0, 0.125), torch.bfloat16, 64)


@pytest.mark.parametrize("dtype,dim,page", [(torch.bfloat16, 64, 16), (torch.float16, 128, 64), (torch.bfloat16, 64, 5), (torch.float32, 32, 16)])
def test_scores_of_minus_infinity(cuda_module, dtype, dim, page):
    """A row that sees only scores of -inf is NaN with lse -inf, in items of one CTA and in ones that several share."""
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    lens = [(1, 3), (9, 5000), (150, 20)]
    q, k, v, table, seq_lens, starts = make_case(lens, 2, 1, dim, page, dtype)
    q.zero_()
    q[..., 0] = -math.inf
    k.fill_(1)
    got = chunk_attention(q, PagedCache(k, v), table, seq_lens, starts).check()
    assert bool(got.out.isnan().all()) and bool((got.lse == -math.inf).all())


def test_append_in_place_and_output_that_is_the_input(cuda_module):
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention, rotary_append
    for dtype, dim in ((torch.bfloat16, 64), (torch.float32, 6)):
        gen = torch.Generator(device="cuda").manual_seed(2)
        q = torch.randn((50, 4, dim), generator=gen, device="cuda").to(dtype)
        k, v = (torch.randn((50, 2, dim), generator=gen, device="cuda").to(dtype) for _ in range(2))
        cos, sin = (torch.randn((64, dim // 2), generator=gen, device="cuda") for _ in range(2))
        cache = PagedCache.allocate(8, 16, 2, dim, dtype=dtype)
        at = torch.arange(50, dtype=torch.int32, device="cuda")
        want = rotary_append(q, k, v, cos, sin, at, at.long(), cache)
        got = rotary_append(q, k, v, cos, sin, at, at.long(), cache, out=q)
        assert got is q and torch.equal(got, want)
        with pytest.raises(RuntimeError, match="must not be q"):
            chunk_attention(q, cache, torch.arange(8, dtype=torch.int32, device="cuda")[None], i32([50]), i32([0, 50]), out=q)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page", [(torch.bfloat16, 16, 8, 64, 16), (torch.float16, 8, 8, 128, 32), (torch.bfloat16, 28, 4, 128, 128)])
@pytest.mark.parametrize("longest", [1, 120, 129, 300, 700])
def test_many_short_sequences(cuda_module, dtype, heads, kv_heads, dim, page, longest):
    """Several items per CTA, most of them of a single key tile, in which one half of the softmax threads has nothing to do."""
    rng = np.random.default_rng(longest)
    lens = [(1, int(x)) for x in rng.integers(0, longest, 260)]
    check_attention(lens, heads, kv_heads, dim, page, dtype)
    mixed = [(int(n), int(x)) for n, x in zip(rng.choice([0, 1, 1, 1, 9, 40, 150], 150), rng.integers(0, longest, 150))]
    check_attention(mixed, heads, kv_heads, dim, page, dtype)
    check_attention(mixed, heads, kv_heads, dim, page, dtype, window=50, sinks=3)


BROKEN = {  # starts, (past, rows in order of the packed step) of the sequences that own rows, statuses
    "beyond": ([0, 3, 1000, 7, 9], [30, 100, 0, 4000], [0, 6, 6, 0]),
    "unordered": ([5, 8, 0, 5], [3000, 10, 700], [0, 6, 0]),
    "overlapping": ([0, 10, 5, 20, 27], [4000, 100, 3000, 500], [6, 6, 6, 0]),
    "inside": ([0, 9, 3, 5, 12], [300, 20, 3000, 40], [6, 6, 6, 6]),
    "negative": ([0, 4, -3, 6, 9], [300, 50, 600, 90], [0, 6, 6, 0]),
    "nested": ([0, 2, 40, 6, 3, 5, 8], [50, 600, 70, 800, 90, 2000], [0, 6, 6, 6, 0, 0]),
}


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 40)])
@pytest.mark.parametrize("kind", list(BROKEN))
def test_starts_broken_in_the_middle(cuda_module, dtype, dim, kind):
    """Row starts out of order or beyond the step: a sequence whose rows lie in the step and are claimed by no other one is computed
    as ever, every other row that some sequence claims is 0 with lse -inf, the rest is left as it was."""
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    starts, past, status = BROKEN[kind]
    seqs, n = len(past), max(x for x in starts if x < 30)
    mine = [max(b - a, 0) if a >= 0 and b <= n else 0 for a, b in zip(starts, starts[1:])]
    lens = [(m, p) for m, p in zip(mine, past)]
    q, k, v, table, seq_lens, _ = make_case([(m, p) for m, p in lens], 4, 2, dim, 16, dtype)
    q = torch.cat((q, q))[:n] if q.shape[0] >= n / 2 else torch.cat([q] * n)[:n]
    out = torch.full((n + 2, 4, dim), 5.0, dtype=dtype, device="cuda")
    got = chunk_attention(torch.cat((q, q[:2])), PagedCache(k, v), table, seq_lens, i32(starts), out=out)
    # `n + 2` rows: a start of 1000 or 40 lies beyond the step, the last two rows behind every sequence that fits.
    assert got.status.tolist() == status
    claimed = torch.zeros(n + 2, dtype=torch.bool, device="cuda")
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        claimed[max(a, 0):max(min(b, n + 2), 0)] = True
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        if status[s]:
            continue
        want = definition(q[a:b], k, v, table[s:s + 1], [lens[s]], 0, 0, dim ** -0.5)
        assert_close(type(got)(got.out[a:b], got.lse[a:b], got.status), want, dtype, dim)
        claimed[a:b] = False
        out[a:b] = 5.0
    assert bool((out[claimed] == 0).all()) and bool((got.lse[claimed] == -math.inf).all())
    assert bool((out[~claimed] == 5).all())


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float32, 8)])
def test_broken_starts_over_many_rows(cuda_module, dtype, dim):
    """A failed sequence that claims more rows than one bitmap holds, around others that own some of them."""
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    n = 140000
    starts = [0, 3, n + 5, 65530, 65560, n + 9, n - 7, n]
    lens = [(3, 20), (0, 5), (0, 5), (30, 50), (0, 5), (0, 5), (7, 40)]
    q, k, v, table, seq_lens, _ = make_case(lens, 1, 1, dim, 16, dtype)
    full = torch.zeros((n, 1, dim), dtype=dtype, device="cuda")
    rows = [slice(0, 3), slice(65530, 65560), slice(n - 7, n)]
    at = 0
    for r in rows:
        full[r] = q[at:at + r.stop - r.start]
        at += r.stop - r.start
    out = torch.full((n, 1, dim), 5.0, dtype=dtype, device="cuda")
    got = chunk_attention(full, PagedCache(k, v), table, seq_lens, i32(starts), out=out)
    assert got.status.tolist() == [0, 6, 6, 0, 6, 6, 0]
    fine = [(0, 3, 0), (65530, 65560, 3), (n - 7, n, 6)]
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    for a, b, s in fine:
        want = definition(full[a:b], k, v, table[s:s + 1], [lens[s]], 0, 0, dim ** -0.5)
        assert_close(type(got)(got.out[a:b], got.lse[a:b], got.status), want, dtype, dim)
        rest[a:b] = False
    assert bool((out[rest] == 0).all()) and bool((got.lse[rest] == -math.inf).all())


@pytest.mark.parametrize("dtype,dim,page", [(torch.bfloat16, 64, 16), (torch.float16, 128, 64)])
def test_waits_that_run_out(cuda_module, dtype, dim, page):
    """Pages that never arrive: the call ends after its limit, every sequence reports status 7, and the next call is right."""
    from bitmask_speculation_b200 import _native
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    lens = [(1, 700), (9, 5000), (300, 900), (1, 3)]
    q, k, v, table, seq_lens, starts = make_case(lens, 8, 2, dim, page, dtype)
    cache = PagedCache(k, v)
    lib = _native.library()
    _native.check(lib.bms_hold_pages(1))
    try:
        held = chunk_attention(q, cache, table, seq_lens, starts)
        torch.cuda.synchronize()
    finally:
        _native.check(lib.bms_hold_pages(0))
    assert held.status.tolist() == [7] * 4
    with pytest.raises(ValueError, match=r"\(1, 7\)"):
        held.check()
    for _ in range(2):
        got = chunk_attention(q, cache, table, seq_lens, starts)
        assert got.status.tolist() == [0] * 4
        assert_close(got, definition(q, k, v, table, lens, 0, 0, dim ** -0.5), dtype, dim)


@pytest.mark.parametrize("dtype,dim,page", [(torch.bfloat16, 64, 16), (torch.float16, 128, 64)])
def test_rows_of_a_call_that_gave_up_are_cleared(cuda_module, dtype, dim, page):
    """No block joins parts of divided items, or computes items again, while another one clears their rows."""
    from bitmask_speculation_b200 import _native
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    lens = [(2000, 300), (150, 6000), (9, 20000), (700, 0)]
    q, k, v, table, seq_lens, starts = make_case(lens, 8, 2, dim, page, dtype)
    k[table[0, 0]] = math.nan
    v[table[1, :20].long()] = math.inf
    cache = PagedCache(k, v)
    out = torch.full((q.shape[0] + 5, 8, dim), 5.0, dtype=dtype, device="cuda")
    padded = torch.cat((q, q[:5]))
    lib = _native.library()
    _native.check(lib.bms_hold_pages(1))
    try:
        for _ in range(3):
            held = chunk_attention(padded, cache, table, seq_lens, starts, out=out)
            assert held.status.tolist() == [7] * 4
            assert bool((out[:-5] == 0).all()) and bool((held.lse[:-5] == -math.inf).all())
            assert bool((out[-5:] == 5).all())
    finally:
        _native.check(lib.bms_hold_pages(0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_positions_near_the_32_bit_end(cuda_module, dtype):
    """A windowed token at the largest position that a table of these pages reaches: it sees what it would see at the end of one
    page, and a page outside the cache is noticed."""
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    page = 511 * 128
    width = (2 ** 31 - 257) // page
    gen = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.randn((2, page, 1, 64), generator=gen, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn((1, 2, 64), generator=gen, device="cuda").to(dtype)
    cache, starts = PagedCache(k, v), i32([0, 1])
    table = torch.zeros((1, width), dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    want = chunk_attention(q, cache, i32([[1]]), i32([page]), starts, window=100).check()
    got = chunk_attention(q, cache, table, i32([width * page]), starts, window=100)
    assert got.status.tolist() == [0] and torch.equal(got.out, want.out) and torch.equal(got.lse, want.lse)
    table[0, -1] = 2
    assert chunk_attention(q, cache, table, i32([width * page]), starts, window=100).status.tolist() == [11]
    assert chunk_attention(q, cache, table, i32([(width - 1) * page]), starts, window=100).status.tolist() == [0]


def test_calls_of_several_threads(cuda_module):
    """Four threads on streams of their own run every operator at once (foreign calls release the interpreter's lock)."""
    from concurrent.futures import ThreadPoolExecutor
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention, plan_pages, rotary_append

    def work(seed):
        results = []
        with torch.cuda.stream(torch.cuda.Stream()):
            gen = torch.Generator(device="cuda").manual_seed(seed)
            for i in range(12):
                dtype, dim = ((torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 32))[i % 3]
                cache = PagedCache.allocate(64, 16, 2, dim, dtype=dtype)
                table = torch.zeros((2, 30), dtype=torch.int32, device="cuda")
                plan = plan_pages(i32([0, 0]), i32([300, 9]), i32([0, 0]), table, torch.arange(64, dtype=torch.int32, device="cuda"), i32([64]),
                                  page_size=16, tokens=309)
                q, k, v = (torch.randn((309, h, dim), generator=gen, device="cuda").to(dtype) for h in (4, 2, 2))
                turned = rotary_append(q, k, v, *rope_tables(320, dim), plan.positions, plan.slots, cache)
                out = chunk_attention(turned, cache, table, plan.seq_lens, plan.query_start).check().out
                x = torch.randn((5, 9001), generator=gen, device="cuda").to(dtype)
                u = torch.rand(5, dtype=torch.float64, generator=gen, device="cuda")
                results.append((out, batched_filtered_sample(x, None, top_p=0.9, uniforms=u).check().token_ids))
            torch.cuda.current_stream().synchronize()
        return results

    want = [work(seed) for seed in range(4)]
    with ThreadPoolExecutor(4) as pool:
        got = list(pool.map(work, range(4)))
    for a, b in zip(want, got):
        for (x, s), (y, t) in zip(a, b):
            assert torch.equal(x, y) and torch.equal(s, t)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("scale", [0.0, 1e-33, -1e-33])
def test_scales_near_zero_of_large_scores(cuda_module, dtype, dim, scale):
    """A scale of 0 weighs all visible keys alike however large the products are; one of 1e-33 is not rounded up to anything."""
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    lens = LENS["round"]
    q, k, v, table, seq_lens, starts = make_case(lens, 4, 2, dim, 16, dtype)
    q, k = q * 2.0 ** 51, k * 2.0 ** 50
    got = chunk_attention(q, PagedCache(k, v), table, seq_lens, starts, scale=scale)
    assert_close(got, definition(q, k, v, table, lens, 0, 0, scale), dtype, dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_captured_round_follows_its_inputs(cuda_module, dtype):
    """Plan, append, attention and sampling captured once: replays with other lengths, tables, values and uniforms equal direct
    calls, on a second stream too."""
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention, plan_pages, rotary_append
    seqs, width, page, n, dim = 3, 40, 16, 420, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda").to(dtype)  # noqa: E731
    cos, sin = rope_tables(width * page, dim)
    state = dict(past=i32([0, 0, 0]), new=i32([400, 9, 1]), held=i32([0] * 3), count=i32([120]), u=torch.rand(seqs, dtype=torch.float64, generator=gen, device="cuda"),
                 q=rand(n, 4, dim), k=rand(n, 2, dim), v=rand(n, 2, dim), x=rand(seqs, 9001))

    def run(s, table, free, cache):
        plan = plan_pages(s["past"], s["new"], s["held"], table, free, s["count"], page_size=page, tokens=n)
        turned = rotary_append(s["q"], s["k"], s["v"], cos, sin, plan.positions, plan.slots, cache)
        out = chunk_attention(turned, cache, table, plan.seq_lens, plan.query_start, window=300, sinks=4)
        return plan, out, batched_filtered_sample(s["x"], None, top_p=0.9, top_k=3000, uniforms=s["u"])

    def fresh():
        return torch.zeros((seqs, width), dtype=torch.int32, device="cuda"), torch.arange(120, dtype=torch.int32, device="cuda"), PagedCache.allocate(120, page, 2, dim, dtype=dtype)

    mine, other = fresh(), fresh()
    warm = fresh()
    run(state, *warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(state, *mine)
    stream = torch.cuda.Stream()
    for i, (past, new) in enumerate([([0, 0, 0], [400, 9, 1]), ([391, 5, 1], [9, 300, 1]), ([0, 305, 2], [200, 0, 9]), ([200, 300, 0], [9, 9, 0])]):
        state["past"].copy_(i32(past)), state["new"].copy_(i32(new))
        for name in ("q", "k", "v", "x"):
            state[name].copy_(rand(*state[name].shape))
        state["u"].uniform_(generator=gen)
        want = run(state, *other)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream if i % 2 else torch.cuda.current_stream()):
            graph.replay()
        torch.cuda.synchronize()
        for a, b in ((held[0].check(), want[0].check()), (held[1].check(), want[1].check()), (held[2].check(), want[2].check())):
            for name in a.__slots__:
                x, y = getattr(a, name), getattr(b, name)
                rows = sum(new) if name in ("out", "lse") else None  # rows behind the last sequence are unspecified
                assert torch.equal(x[:rows], y[:rows]), (i, name)
        assert torch.equal(mine[0], other[0]) and torch.equal(mine[1], other[1]) and torch.equal(mine[2].k, other[2].k) and torch.equal(mine[2].v, other[2].v)
        state["held"].copy_(want[0].held), state["count"].copy_(want[0].free_count)


@pytest.mark.parametrize("dtype,dim,page", [(torch.bfloat16, 64, 16), (torch.float16, 128, 64), (torch.float16, 64, 24), (torch.float32, 32, 16)])
def test_scores_that_are_not_finite(cuda_module, dtype, dim, page):
    """Keys whose scores are -inf weigh nothing; a row that sees one of +inf or NaN is NaN, and no other row is."""
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention
    lens = [(1, 300), (9, 6000), (200, 150), (3, 2), (40, 700)]
    for window, sinks in ((0, 0), (90, 3)):
        q, k, v, table, seq_lens, starts = make_case(lens, 4, 2, dim, page, dtype, poison=False)
        q[..., 0] = 1.0
        gen = torch.Generator().manual_seed(dim)
        bad, low = {}, {}
        for s, (n, past) in enumerate(lens):
            for what, count in ((low, 5), (bad, 1 if n > 3 else 0)):
                what[s] = torch.randint(past + (n // 2 if what is bad else 0), past + n, (count,), generator=gen).tolist()
            for i, j in enumerate(low[s] + bad[s]):
                pg = int(table[s, j // page])
                k[pg, j % page, :, 0] = -math.inf if j not in bad[s] else (math.inf if s % 2 else math.nan)
        got = chunk_attention(q, PagedCache(k, v), table, seq_lens, starts, window=window, sinks=sinks).check()
        row = 0
        for s, (n, past) in enumerate(lens):
            at = torch.arange(n + past, device="cuda")
            pg = table[s].long()[at // page]
            ks, vs = k[pg, at % page].double(), v[pg, at % page].double()
            age = (past + torch.arange(n, device="cuda"))[:, None] - at
            seen = age >= 0
            if window:
                seen &= (age < window) | (at < sinks)
            for h in range(4):
                score = q[row:row + n, h].double() @ torch.nan_to_num(ks[:, h // 2], nan=0, posinf=0, neginf=0).T
                extra = torch.where(torch.isfinite(ks[:, h // 2, 0]), 0.0, ks[:, h // 2, 0])
                score = ((score + extra) * dim ** -0.5).masked_fill(~seen, -math.inf)
                want = torch.softmax(score, 1) @ vs[:, h // 2]
                broken = (~(score < math.inf)).any(1)
                mine, lse = got.out[row:row + n, h].double(), got.lse[row:row + n, h]
                assert torch.equal(torch.isnan(mine).all(1), torch.isnan(want).all(1)) and torch.equal(torch.isnan(mine).any(1), torch.isnan(want).any(1))
                assert torch.equal(torch.isnan(lse), broken)
                # Weights and result rounded once each, scores of a few units good to 2^-15 (dim + 4 roundings of 2^-24 of terms below 2^2).
                eps = EPS[dtype] / 2
                weight = torch.softmax(score, 1) @ vs[:, h // 2].abs()
                off = (mine - want).abs()[~broken & ~torch.isnan(want).any(1)]
                assert bool((off <= ((2 * eps + 2.0 ** -14) * weight + 2.0 ** -20)[~broken & ~torch.isnan(want).any(1)]).all())
            row += n
