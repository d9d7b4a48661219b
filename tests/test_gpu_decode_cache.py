"""Decoders over the paged cache: the logits of every call equal those of a full forward, whatever the calls before it
left in the pages, and the request loops choose the same tokens."""

import copy

import pytest

from bitmask_speculation_b200 import workloads as wl

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

VOCAB = 1000


def decoder(dtype, *, layers=2, dim=256, heads=4, kv_heads=2, seed=3, device="cuda", vocab=VOCAB):
    from bitmask_speculation_b200.decode import build_decoder
    return build_decoder(vocab, layers=layers, dim=dim, heads=heads, kv_heads=kv_heads, dtype=dtype, device=device, seed=seed)


def bound(model, want):
    """What a 2-block forward may lose.  A value passes 7 roundings of depth per block (two norms, three projections of up to
    768 terms accumulated in float32, attention, the gate) and three behind the blocks, each at most half a step of its
    own magnitude; norms and residuals keep magnitudes within a few times the output's, so that 2 * 7 + 3 steps of the
    largest logit, with a factor of 2 for both forms, are not reached.  The float32 form adds its accumulations:
    768 terms lose at most 768 half steps, in practice their root (28): 32 covers it."""
    eps = torch.finfo(model.head.weight.dtype).eps / 2
    return 2 * 17 * eps * (32 if model.head.weight.dtype == torch.float32 else 1) * float(want.abs().max())


@pytest.mark.parametrize("dtype,page,dims", [(torch.float32, 16, (256, 4, 2)), (torch.bfloat16, 64, (256, 4, 2)), (torch.bfloat16, 16, (256, 2, 1)),
                                             (torch.float16, 5, (192, 6, 6)), (torch.bfloat16, 32, (128, 8, 1))])
def test_cached_logits_equal_full_forwards(cuda_module, dtype, page, dims):
    """Growing, repeated, shrunk and diverging prefixes, single tokens and long chunks in one sequence."""
    dim, heads, kv_heads = dims
    model = decoder(dtype, dim=dim, heads=heads, kv_heads=kv_heads)
    cached = decoder(dtype, dim=dim, heads=heads, kv_heads=kv_heads).enable_cache(300, page_size=page)
    exact = copy.deepcopy(model).double()
    gen = torch.Generator().manual_seed(5)
    base = torch.randint(0, VOCAB, (300,), generator=gen).tolist()
    other = torch.randint(0, VOCAB, (300,), generator=gen).tolist()
    calls = [(base[:1], 0, 1), (base[:40], 39, 1), (base[:49], 40, 9), (base[:44] + other[:5], 43, 6), (base[:44] + other[:5], 43, 6),
             (base[:44] + other[:6], 49, 1), (base[:64], 60, 4), (base[:65], 64, 1), (other[:200], 0, 200), (base[:10], 9, 1),
             (base, 290, 10), (base[:299] + [7], 299, 1)]
    for tokens, first, rows in calls:
        got = cached.logits(tokens, first, rows)
        want = exact.logits(tokens, first, rows)
        plain = model.logits(tokens, first, rows)
        assert got.shape == (rows, VOCAB)
        limit = bound(model, want)
        assert float((plain.double() - want).abs().max()) <= limit
        assert float((got.double() - want).abs().max()) <= limit, (len(tokens), first)
    assert int(cached._cache.free_count) == cached._cache.free_pages.shape[0] - int(cached._cache.held.sum())


def test_batches_of_sequences_share_a_forward(cuda_module):
    """Sequences of different lengths in one call; one that leaves gives its pages back and may come again."""
    model, cached = decoder(torch.bfloat16), decoder(torch.bfloat16).enable_cache(200, sequences=3, page_size=16)
    exact = copy.deepcopy(model).double()
    gen = torch.Generator().manual_seed(6)
    a, b, c = (torch.randint(0, VOCAB, (200,), generator=gen).tolist() for _ in range(3))
    for batch in ([(a[:150], 149, 1), (b[:3], 0, 3), (c[:80], 70, 10)], [(a[:159], 150, 9), (b[:4], 3, 1), (c[:76] + a[:9], 75, 10)],
                  [(a[:160], 159, 1)], [(a[:161], 159, 2), (b[:200], 199, 1)]):
        sequences, firsts, rows = zip(*batch)
        got = cached.logits_batch(sequences, firsts, rows)
        for g, (tokens, first, n) in zip(got, batch):
            want = exact.logits(tokens, first, n)
            assert g.shape == want.shape and float((g.double() - want).abs().max()) <= bound(model, want)
    assert cached._cache.held.tolist() == [11, 13, 0]
    with pytest.raises(ValueError):
        cached.logits_batch([a[:5]] * 4, [0] * 4, [1] * 4)
    with pytest.raises(ValueError):
        cached.logits_batch([a + [1]], [0], [1])
    with pytest.raises(ValueError):
        cached.logits_batch([a[:5]], [5], [1])
    with pytest.raises(ValueError):
        model.logits_batch([a[:5]], [4], [1])


def test_request_loops_over_the_cache_choose_the_same_tokens(cuda_module):
    from bitmask_speculation_b200.decode import constrained_greedy, random_prompts, speculative_c4
    vocab = 8320
    make = lambda: (decoder(torch.float32, dim=256, seed=1, vocab=vocab), decoder(torch.float32, layers=1, dim=128, heads=2, kv_heads=1, seed=2, vocab=vocab))
    target, draft = make()
    c_target, c_draft = make()
    c_target.enable_cache(128, page_size=16), c_draft.enable_cache(128, page_size=16)
    for i, prompt in enumerate(random_prompts(4, 16, vocab, seed=3)):
        g0 = wl.SyntheticDFAGrammar(vocab, states=64, seed=10 + i)
        want = constrained_greedy(target, prompt, g0.fork(), max_new_tokens=48, eos=(0,))
        got = constrained_greedy(c_target, prompt, g0.fork(), max_new_tokens=48, eos=(0,))
        assert (got.token_ids, got.stop_reason) == (want.token_ids, want.stop_reason), i
        spec = speculative_c4(target, draft, prompt, g0.fork(), max_new_tokens=48, eos=(0,))
        c_spec = speculative_c4(c_target, c_draft, prompt, g0.fork(), max_new_tokens=48, eos=(0,))
        assert c_spec == spec, i


def test_sequences_without_rows(cuda_module):
    """Row counts of 0: the forward fills the pages, and gives no logits of those sequences."""
    cached, exact = decoder(torch.bfloat16).enable_cache(100, sequences=2, page_size=16), decoder(torch.bfloat16).double()
    a, b = list(range(40)), list(range(100, 130))
    none = cached.logits_batch([a, b], [39, 29], [0, 0])
    assert [tuple(g.shape) for g in none] == [(0, VOCAB)] * 2
    some = cached.logits_batch([a + [7], b], [40, 29], [1, 0])
    want = exact.logits(a + [7], 40, 1)
    assert some[1].shape == (0, VOCAB) and float((some[0].double() - want).abs().max()) <= bound(cached, want)


def test_changed_weights_forget_the_pages(cuda_module):
    """Keys and values of other weights are not attended to: a changed parameter makes the next call forward the whole prefix."""
    model, cached = decoder(torch.bfloat16), decoder(torch.bfloat16).enable_cache(200, page_size=16)
    other = decoder(torch.bfloat16, seed=9)
    tokens = torch.randint(0, VOCAB, (120,), generator=torch.Generator().manual_seed(7)).tolist()
    cached.logits(tokens[:100], 99, 1)
    changes = (lambda m: m.load_state_dict(other.state_dict()), lambda m: m.blocks[0].kv.weight.mul_(-1.5),
               lambda m: setattr(m.blocks[1].q, "weight", torch.nn.Parameter(m.blocks[1].q.weight.detach().roll(1, 0))),
               lambda m: m.embed.weight.detach().neg_(),
               lambda m: setattr(m.blocks[0], "o", copy.deepcopy(other.blocks[1].o)))
    for i, change in enumerate(changes):
        with torch.no_grad():
            change(model), change(cached)
        n = 101 + i
        want = copy.deepcopy(model).double().logits(tokens[:n], n - 1, 1)
        got = cached.logits(tokens[:n], n - 1, 1)
        assert float((got.double() - want).abs().max()) <= bound(model, want), i
