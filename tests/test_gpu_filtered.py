"""Filtered sampling (temperature, top-k, top-p, min-p under grammar masks) against the definition in
float64 on the host.  Tokens, kept counts and statuses are whole numbers and have to be equal: both
sides weigh and sum in float64, so they could differ only where a uniform or a filter's limit lies
within about 1e-13 of a boundary, which no seeded case here does."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = ("float32", "bfloat16", "float16")


def pack(valid: np.ndarray) -> np.ndarray:
    rows, vocab = valid.shape
    padded = np.zeros((rows, (vocab + 31) // 32 * 32), dtype=bool)
    padded[:, :vocab] = valid
    return np.packbits(padded, axis=1, bitorder="little").view(np.int32)


def definition(x, valid, t, k, p, floor, u):
    """(token, kept, status) of one row of float64 values."""
    if not (0 <= t < np.inf) or not (0 < p <= 1) or not (0 <= floor <= 1) or k < 0:
        return -1, 0, 10
    if np.isnan(x).any():
        return -1, 0, 2
    ids = np.flatnonzero(valid)
    if t > 0 and ids.size and np.isposinf(x[ids]).any():
        return -1, 0, 5
    if ids.size == 0:
        return -1, 0, 1
    if t == 0:
        return int(ids[np.argmax(x[ids])]), 1, 0
    ids = ids[x[ids] > -np.inf]
    if ids.size == 0:
        return -1, 0, 4
    if not 0 <= u < 1:
        return -1, 0, 3
    ids = ids[np.lexsort((ids, -x[ids]))]
    if k:
        ids = ids[:k]
    with np.errstate(over="ignore", under="ignore"):
        w = np.exp((x[ids] - x[ids[0]]) * min(1.0 / t, np.finfo(np.float64).max))
    n = ids.size
    if p < 1:
        before = np.concatenate(([0.0], np.cumsum(w)[:-1]))
        n = int((before < p * w.sum()).sum())
    n = min(n, int((w >= floor).sum()))
    order = np.argsort(ids[:n])
    ids, w = ids[:n][order], w[:n][order]
    c = np.cumsum(w)
    hit = np.flatnonzero((c > u * c[-1]) | (c >= c[-1]))
    return int(ids[hit[0]]), n, 0


def check(values, valid, dtype, params, uniforms, *, mask=True, offset=0, mask_rows=None):
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    rows, vocab = values.shape
    store = torch.empty(rows * vocab + offset, dtype=getattr(torch, dtype), device="cuda")
    logits = store[offset:].view(rows, vocab)  # the base address is offset elements past an aligned one
    logits.copy_(torch.from_numpy(values))
    got = batched_filtered_sample(logits, torch.from_numpy(pack(valid)).cuda() if mask else None, uniforms=torch.from_numpy(uniforms).cuda(),
                                  mask_rows=None if mask_rows is None else torch.tensor(mask_rows, dtype=torch.int32).cuda(), **params)
    exact = logits.double().cpu().numpy()
    per_row = {}
    for name, off in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)):
        v = params.get(name, off)
        per_row[name] = v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(rows, v, dtype=np.float64)
    want = [definition(exact[r], valid[r if mask_rows is None else mask_rows[r]], per_row["temperature"][r], int(per_row["top_k"][r]), per_row["top_p"][r],
                       per_row["min_p"][r], uniforms[r]) for r in range(rows)]
    assert got.status.tolist() == [w[2] for w in want]
    assert got.kept_counts.tolist() == [w[1] for w in want]
    assert got.token_ids.tolist() == [w[0] for w in want]
    return got


FILTERS = (dict(), dict(top_k=1), dict(temperature=0.7, top_k=50, top_p=0.95), dict(top_p=0.9), dict(temperature=1.3, min_p=0.05),
           dict(temperature=0.0), dict(top_k=7000, top_p=0.99), dict(top_k=3000, top_p=0.5, min_p=0.01), dict(temperature=5.0, top_p=0.999),
           dict(top_p=1e-9), dict(min_p=1.0), dict(top_k=10 ** 12))


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 500, 5003, 50257])
@pytest.mark.parametrize("dtype", DTYPES)
def test_filters_over_vocabularies(cuda_module, dtype, vocab):
    rng = np.random.default_rng(vocab)
    for i, params in enumerate(FILTERS):
        rows = 5
        values = (rng.standard_normal((rows, vocab)) * rng.uniform(0.5, 4.0, (rows, 1))).astype(np.float32)
        valid = rng.random((rows, vocab)) < np.array([1.0, 0.7, 0.1, 0.01, 1.0])[:, None]
        valid[:, rng.integers(vocab)] = True
        check(values, valid, dtype, params, rng.random(rows), offset=i % 9)


@pytest.mark.parametrize("rows", [1, 3, 40, 200])
def test_rows_and_clusters(cuda_module, rows):
    """Few rows spread over clusters of CTAs, many rows take one CTA each: the results are the same."""
    rng = np.random.default_rng(rows)
    vocab = 20011
    values = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    valid = rng.random((rows, vocab)) < rng.random((rows, 1))
    valid[:, 17] = True
    for params in (dict(top_k=40, top_p=0.9), dict(top_p=0.8), dict(min_p=0.1), dict()):
        check(values, valid, "bfloat16", params, rng.random(rows))


def test_rows_bring_their_own_parameters(cuda_module):
    rng = np.random.default_rng(4)
    rows, vocab = 64, 9001
    pick = lambda choices, dtype: torch.tensor(rng.choice(choices, rows), dtype=dtype, device="cuda")  # noqa: E731
    params = dict(temperature=pick([0.0, 0.5, 1.0, 2.0], torch.float32), top_k=pick([0, 1, 5, 100, 6000, 2 ** 31 - 1], torch.int32),
                  top_p=pick([1.0, 0.9, 0.5], torch.float32), min_p=pick([0.0, 0.1, 1.0], torch.float32))
    values = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    valid = rng.random((rows, vocab)) < 0.8
    for dtype in DTYPES:
        check(values, valid, dtype, params, rng.random(rows))
    # Numbers and tensors mix.
    check(values, valid, "float16", dict(params, top_p=0.7, temperature=1.0), rng.random(rows))


def test_bad_row_parameters_fail_their_rows_only(cuda_module):
    rng = np.random.default_rng(5)
    nan, inf = float("nan"), float("inf")
    t = torch.tensor([1.0, -1.0, nan, inf, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0], dtype=torch.float32, device="cuda")
    k = torch.tensor([3, 3, 3, 3, -1, 3, 3, 3, 3, 3], dtype=torch.int32, device="cuda")
    p = torch.tensor([0.5, 0.5, 0.5, 0.5, 0.5, 0.0, nan, 1.5, 0.5, 0.5], dtype=torch.float32, device="cuda")
    m = torch.tensor([0.1, 0.1, 0.1, 0.1, 0.1, 0.1, 0.1, 0.1, -0.1, nan], dtype=torch.float32, device="cuda")
    got = check(rng.standard_normal((10, 300)).astype(np.float32), np.ones((10, 300), dtype=bool), "float32",
                dict(temperature=t, top_k=k, top_p=p, min_p=m), rng.random(10))
    assert got.status.tolist() == [0] + [10] * 9
    with pytest.raises(ValueError, match="status"):
        got.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lowest_token(cuda_module, dtype):
    """Scores of few distinct values: the cut of every filter falls inside a run of equal scores, in
    the list path (small rows) and in the bisected one."""
    rng = np.random.default_rng(6)
    for vocab in (64, 3001, 12007):
        values = rng.integers(-3, 3, (6, vocab)).astype(np.float32)
        valid = rng.random((6, vocab)) < 0.9
        valid[:, 0] = True
        for params in (dict(top_k=17), dict(top_k=vocab * 2 // 3), dict(top_p=0.6), dict(top_p=0.97), dict(top_k=vocab // 2, top_p=0.5)):
            check(values, valid, dtype, params, rng.random(6))


@pytest.mark.parametrize("vocab", [10, 4096, 4097, 30000])
def test_equal_scores(cuda_module, vocab):
    rng = np.random.default_rng(7)
    values = np.full((3, vocab), -1.5, dtype=np.float32)
    values[1] = 0.0
    values[1, ::2] = -0.0  # ranks with +0
    valid = np.ones((3, vocab), dtype=bool)
    for params in (dict(top_p=0.3), dict(top_k=vocab - 1), dict(min_p=1.0), dict()):
        check(values, valid, "float32", params, rng.random(3))


def test_masked_infinities_and_nan_rows(cuda_module):
    rng = np.random.default_rng(8)
    for vocab in (700, 9000):
        values = rng.standard_normal((9, vocab)).astype(np.float32)
        valid = rng.random((9, vocab)) < 0.6
        valid[:, 5] = True
        values[0][~valid[0]] = np.inf  # masked +inf does not count
        values[1, 5] = np.inf
        values[2, int(np.flatnonzero(~valid[2])[0])] = np.nan  # NaN anywhere fails the row
        valid[3] = False
        values[4][valid[4]] = -np.inf
        values[5, ::2] = -np.inf
        values[6] = np.finfo(np.float32).min  # the type's lowest value is a score like any other
        values[7] = np.finfo(np.float32).min
        values[7, 5] = np.finfo(np.float32).max
        values[8][valid[8]] = -np.inf
        values[8, 5] = -3.0
        for params in (dict(), dict(top_k=4, top_p=0.5), dict(top_p=0.9), dict(min_p=0.2), dict(temperature=0.0)):
            check(values, valid, "float32", params, rng.random(9))


def test_uniforms_and_temperatures_at_their_ends(cuda_module):
    rng = np.random.default_rng(9)
    for vocab in (300, 8000):
        values = rng.standard_normal((6, vocab)).astype(np.float32)
        valid = rng.random((6, vocab)) < 0.7
        valid[:, 2] = True
        u = np.array([0.0, 1.0 - 2.0 ** -53, -0.1, 1.0, np.nan, 0.5])
        for t in (1e-300, 1e-3, 1.0, 1e300):
            for params in (dict(), dict(top_k=5), dict(top_p=0.9), dict(min_p=0.5)):
                check(values, valid, "float32", dict(params, temperature=t), u)


def test_mask_table_and_no_mask(cuda_module):
    rng = np.random.default_rng(10)
    values = rng.standard_normal((5, 6000)).astype(np.float32)
    table = rng.random((3, 6000)) < 0.5
    check(values, table, "bfloat16", dict(top_p=0.9), rng.random(5), mask_rows=[2, 0, 0, 1, 2])
    check(values, np.ones((5, 6000), dtype=bool), "bfloat16", dict(top_k=30), rng.random(5), mask=False)
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    got = batched_filtered_sample(torch.from_numpy(values).cuda(), torch.from_numpy(pack(table)).cuda(), top_k=3,
                                  mask_rows=torch.tensor([0, 3, -1, 1, 2], dtype=torch.int32, device="cuda"))
    assert got.status.tolist() == [0, 8, 8, 0, 0] and got.token_ids[1:3].tolist() == [-1, -1]


def test_padding_bits_are_ignored(cuda_module):
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    x = torch.zeros((2, 33), device="cuda")
    mask = torch.full((2, 2), -1, dtype=torch.int32, device="cuda")
    assert batched_filtered_sample(x, mask, top_p=0.999).kept_counts.tolist() == [33, 33]


def test_filters_off_agrees_with_the_masked_sampler(cuda_module):
    from bitmask_speculation_b200 import workloads as wl
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    import oracle
    bits, masks, uniforms, temperature = wl.sample_config_np(seed=2, vocab=8192)
    logits = torch.from_numpy(bits.view(np.int16)).view(torch.float16).cuda()
    got = batched_filtered_sample(logits, torch.from_numpy(masks).cuda(), temperature=temperature, uniforms=torch.from_numpy(uniforms).cuda())
    tokens, status = oracle.sample_rows(bits, masks, temperature, uniforms, dtype="float16")
    assert got.status.tolist() == status.tolist()
    for r, (g, e) in enumerate(zip(got.token_ids.tolist(), tokens.tolist())):
        assert oracle.sample_matches(oracle.widen(bits[r], "float16"), masks[r], temperature, uniforms[r], g, e)


def test_streams_graphs_and_empty_batches(cuda_module):
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    rng = np.random.default_rng(11)
    x = torch.from_numpy(rng.standard_normal((4, 7000)).astype(np.float32)).cuda()
    u = torch.from_numpy(rng.random(4)).cuda()
    call = lambda: batched_filtered_sample(x, None, top_p=0.8, top_k=2000, uniforms=u)  # noqa: E731
    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    side.synchronize()
    assert other.token_ids.tolist() == want.token_ids.tolist()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for _ in range(2):
        u.copy_(torch.from_numpy(rng.random(4)))
        graph.replay()
        again = call()
        assert held.token_ids.tolist() == again.token_ids.tolist() and held.kept_counts.tolist() == again.kept_counts.tolist()
    empty = batched_filtered_sample(x[:0], None, top_k=3)
    assert empty.token_ids.shape == (0,)


def test_draws_follow_the_filtered_softmax(cuda_module):
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    from scipy.stats import chisquare
    gen = torch.Generator(device="cuda").manual_seed(3)
    row = torch.randn(200, generator=gen, device="cuda")
    n = 20000
    got = batched_filtered_sample(row.expand(n, 200).contiguous(), None, temperature=0.8, top_k=12, generator=gen)
    p = torch.softmax(row.double() / 0.8, 0)
    top = torch.topk(p, 12).indices
    assert set(got.token_ids.unique().tolist()) <= set(top.tolist())
    counts = torch.bincount(got.token_ids, minlength=200)[top].cpu().numpy()
    want = (p[top] / p[top].sum()).cpu().numpy() * n
    assert chisquare(counts, want).pvalue > 1e-4


def test_refusals(cuda_module):
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample as call
    x = torch.zeros((2, 64), device="cuda")
    mask = torch.full((2, 2), -1, dtype=torch.int32, device="cuda")
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_p=0.0), dict(top_p=1.5), dict(min_p=-0.1), dict(top_k=-1)):
        with pytest.raises(ValueError):
            call(x, mask, **bad)
    for bad in (dict(temperature="1"), dict(top_k=1.5), dict(top_p=True), dict(top_k=torch.ones(2, device="cuda")), dict(top_p=torch.ones(2, device="cuda").double())):
        with pytest.raises(TypeError):
            call(x, mask, **bad)
    with pytest.raises(ValueError):
        call(x, mask, top_p=torch.ones(3, device="cuda"))
    with pytest.raises(ValueError):
        call(x, mask, top_p=torch.ones(2))
    with pytest.raises(ValueError):
        call(x, mask[:1])
    with pytest.raises(ValueError):
        call(x.t(), None)
    with pytest.raises(ValueError):
        call(x, None, mask_rows=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError):
        call(x.double(), mask)


SPREADS = {
    "tiny": lambda rng, n: rng.standard_normal(n) * 1e-3,
    "zeros": lambda rng, n: rng.choice([0.0, -0.0, 1e-4, -1e-4, 0.5, -0.5], n),
    "around_zero": lambda rng, n: rng.standard_normal(n) * 0.02,
    "negative": lambda rng, n: rng.standard_normal(n) * 2 - 40,
    "just_negative": lambda rng, n: -np.abs(rng.standard_normal(n)) * 0.3 - 0.001,
    "high": lambda rng, n: rng.standard_normal(n) * 0.6 + 100,
    "coarse": lambda rng, n: np.round(rng.standard_normal(n) * 2),
    "wide": lambda rng, n: rng.standard_normal(n) * 10.0 ** rng.uniform(-6, 4, n),
    "outlier": lambda rng, n: np.where(np.arange(n) == n // 2, 3e4, rng.standard_normal(n) * 3),
}


@pytest.mark.parametrize("rows", [6, 150, 700])
@pytest.mark.parametrize("spread", list(SPREADS))
def test_spreads_of_scores(cuda_module, spread, rows):
    """Rows beyond the list path whose filters end near zero, far below the maximum, among equal scores, on either side of
    zero; with one CTA per row and with several."""
    rng = np.random.default_rng(rows + len(spread))
    vocab = 9973 if rows > 6 else 40009
    values = SPREADS[spread](rng, rows * vocab).reshape(rows, vocab).astype(np.float32)
    valid = rng.random((rows, vocab)) < rng.choice([1.0, 0.85, 0.6], rows)[:, None]
    valid[:, 5] = True
    scale = {"wide": 3e3, "outlier": 2e4, "high": 0.5}.get(spread, 1.0)
    cases = (dict(top_p=0.31371), dict(top_p=0.90713), dict(top_p=0.99931, temperature=7.0 * scale), dict(top_k=5003, temperature=scale),
             dict(top_k=vocab // 2, top_p=0.70717, temperature=2 * scale), dict(top_p=0.93711, min_p=0.03, temperature=scale))
    for i, params in enumerate(cases if rows < 700 else cases[1:5:2]):
        for dtype in DTYPES if rows == 6 else ("bfloat16",):
            check(values, valid, dtype, params, rng.random(rows), offset=3 * i)


@pytest.mark.parametrize("spread", list(SPREADS))
def test_spreads_of_short_rows(cuda_module, spread):
    """The same spreads in rows, and sparse masks of longer rows, that fit the list of 4,096 tokens."""
    rng = np.random.default_rng(len(spread))
    scale = {"wide": 3e3, "outlier": 2e4, "high": 0.5}.get(spread, 1.0)
    for rows, vocab, density in ((40, 3001, (1.0, 0.7, 0.3)), (9, 60013, (0.06, 0.03, 0.012))):
        values = SPREADS[spread](rng, rows * vocab).reshape(rows, vocab).astype(np.float32)
        valid = rng.random((rows, vocab)) < rng.choice(density, rows)[:, None]
        valid[:, 5] = True
        for i, params in enumerate((dict(top_p=0.31371), dict(top_p=0.99931, temperature=7.0 * scale), dict(top_k=703, temperature=scale),
                                    dict(top_k=1511, top_p=0.70717, temperature=2 * scale), dict(top_p=0.93711, min_p=0.03, temperature=scale))):
            for dtype in DTYPES:
                check(values, valid, dtype, params, rng.random(rows), offset=3 * i)


@pytest.mark.parametrize("vocab", [8192, 16385, 32771])
def test_clusters_that_start_while_others_end(cuda_module, vocab):
    """Rows of the shortest parts that a cluster of 2, 4 or 8 CTAs takes, launched back to back on two streams: a CTA may be done
    with its part before another one of its cluster has started."""
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    rng = np.random.default_rng(vocab)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rows in (3, 9, 74, 150):
        values = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
        valid = rng.random((rows, vocab)) < rng.choice([1.0, 0.3, 0.002], rows)[:, None]
        valid[:, rng.integers(vocab)] = True
        u = rng.random(rows)
        params = dict(top_k=40, top_p=0.9)
        want = check(values, valid, "bfloat16", params, u)
        args = torch.from_numpy(values).cuda().bfloat16(), torch.from_numpy(pack(valid)).cuda()
        uniforms = torch.from_numpy(u).cuda()
        torch.cuda.synchronize()
        got = []
        for i in range(40):
            with torch.cuda.stream(streams[i % 2]):
                got.append(batched_filtered_sample(*args, uniforms=uniforms, **params))
        torch.cuda.synchronize()
        for g in got:
            assert torch.equal(g.token_ids, want.token_ids) and torch.equal(g.kept_counts, want.kept_counts) and int(g.status.sum()) == 0


@pytest.mark.parametrize("vocab", [9973, 40009])
def test_min_p_between_zero_and_the_first_bin(cuda_module, vocab):
    """bfloat16 rows whose maximum lies within 2^-7 of zero and whose nucleus ends behind it, while min-p keeps only scores nearer
    to zero than 2^-7: scores of exactly -2^-7 are dropped, in the middle of the row and at its ends alike."""
    rng = np.random.default_rng(vocab)
    u = np.array([0.0, 1e-9, 0.1, 0.5, 0.9, 0.999999])
    for offset in range(9):
        values = rng.choice([-2.0 ** -7, -0.010009765625, -0.0125732421875], (6, vocab)).astype(np.float32)
        values[:, :9] = values[:, -9:] = -2.0 ** -7
        values[np.arange(6)[:, None], rng.integers(9, vocab - 9, (6, 5))] = -0.00099945068359375
        for params in (dict(top_p=0.93, min_p=0.999), dict(top_k=vocab * 3 // 4, min_p=0.999), dict(top_k=vocab * 3 // 4, top_p=0.93, min_p=1.0)):
            got = check(values, np.ones((6, vocab), dtype=bool), "bfloat16", params, u, offset=offset)
            assert max(got.kept_counts.tolist()) <= 5


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_far_below_the_maximum_are_drawn(cuda_module, dtype):
    """A nucleus that reaches weights of 4e-16 of the largest, which lie in the lowest tokens by themselves: a uniform of 0 draws the
    first of them.  min-p ends what is kept above 2e-16, so that the rounding of sums near 1 decides nothing."""
    vocab = 5001
    rng = np.random.default_rng(3)
    values = np.empty((3, vocab), dtype=np.float32)
    values[:, :500] = -35.5
    values[:, 500:3500] = -36.25
    values[:, 3500:] = np.float32(rng.uniform(-12.5, -11.5, (3, vocab - 3500))).astype(np.float16)
    values[:, 4000] = 0.0
    got = check(values, np.ones((3, vocab), dtype=bool), dtype, dict(top_p=1.0 - 3e-13, min_p=3e-16), np.array([0.0, 0.5, 0.9999]))
    assert got.token_ids[0].item() == 0 and got.kept_counts[0].item() == 500 + 1501


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_in_batches_of_every_size(cuda_module, dtype):
    """One row's draws in batches that give it 8, 4, 2 and 1 CTAs, twice each: the same tokens and counts."""
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    gen = torch.Generator(device="cuda").manual_seed(8)
    vocab = 40009
    others = (torch.randn((700, vocab), generator=gen, device="cuda") * 2).to(getattr(torch, dtype))
    row = others[0].clone()
    u = torch.rand(700, dtype=torch.float64, generator=gen, device="cuda")
    for params in (dict(top_k=40, top_p=0.9), dict(top_p=0.8), dict(top_p=0.999, temperature=2.0), dict(min_p=0.1), dict(top_k=9000, top_p=0.95), dict()):
        want = None
        for rows in (1, 3, 40, 200, 700):
            for at in {0, rows // 2, rows - 1}:
                x, un = others[:rows].clone(), u[:rows].clone()
                x[at], un[at] = row, 0.37123
                for _ in range(2):
                    got = batched_filtered_sample(x, None, uniforms=un, **params)
                    one = int(got.token_ids[at]), int(got.kept_counts[at]), int(got.status[at])
                    want = want or one
                    assert one == want, (params, rows, at)
