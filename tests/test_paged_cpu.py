"""Refusals of the paged-cache operators and the filtered sampler that need no GPU: the C entry points turn bad
arguments away before they touch a device, the Python calls before they load the library."""

import ctypes

import pytest

from bitmask_speculation_b200 import _native
from bitmask_speculation_b200.build import build

torch = pytest.importorskip("torch")
INVALID, UNSUPPORTED = _native.ERROR_INVALID_ARGUMENT, _native.ERROR_UNSUPPORTED
PTR = ctypes.c_void_p(256)  # never dereferenced: every call below is refused first


@pytest.fixture(scope="module")
def lib():
    build()
    return _native.library()


def pair(*x):
    return (ctypes.c_int64 * 2)(*x)


def cache(**change):
    shape = dict(pages=4, page_size=16, kv_heads=2, dim=64)
    shape.update({k: v for k, v in change.items() if k in shape})
    strides = change.get("strides", (2048, 128, 64))
    triple = ctypes.c_int64 * 3
    return _native.Cache(256, 256, *shape.values(), triple(*strides), triple(*strides))


# ---------------------------------------------------------------- C entry points
def test_filtered_sample_refusals(lib):
    def call(dtype=0, rows=1, vocab=32, temperature=1.0, top_p=1.0, min_p=0.0, top_k=0, masks=None, mask_rows=None, table=0, filt=True):
        f = _native.Filter(temperature, top_p, min_p, top_k)
        return lib.bms_filtered_sample_batch(PTR, dtype, masks, mask_rows, table, rows, vocab, ctypes.byref(f) if filt else None, PTR, PTR, PTR, PTR, 0, None)
    nan, inf = float("nan"), float("inf")
    for bad in (dict(dtype=3), dict(dtype=-1), dict(vocab=0), dict(vocab=2 ** 31), dict(rows=-1), dict(filt=False), dict(temperature=-0.5), dict(temperature=nan),
                dict(temperature=inf), dict(top_p=0.0), dict(top_p=1.5), dict(top_p=nan), dict(min_p=-0.1), dict(min_p=1.1), dict(min_p=nan),
                dict(top_k=-1), dict(mask_rows=PTR)):
        assert call(**bad) == INVALID, bad
        assert lib.bms_last_error()
    assert call(vocab=2 ** 31 - 1) == UNSUPPORTED


def test_page_plan_refusals(lib):
    def call(seqs=2, width=4, pages=8, page=16, tokens=4):
        return lib.bms_page_plan(PTR, PTR, PTR, seqs, PTR, width, PTR, pages, PTR, page, tokens, PTR, PTR, PTR, PTR, PTR, PTR, PTR, 0, None)
    for bad in (dict(seqs=0), dict(seqs=-1), dict(width=0), dict(pages=0), dict(page=0), dict(page=-16), dict(tokens=-1)):
        assert call(**bad) == INVALID, bad
    for bad in (dict(seqs=8193), dict(pages=2 ** 30), dict(page=65537), dict(tokens=2 ** 30), dict(width=2 ** 30), dict(width=2 ** 28, page=16)):
        assert call(**bad) == UNSUPPORTED, bad


def test_rotary_append_refusals(lib):
    def call(dtype=1, tokens=3, heads=4, qs=pair(256, 64), max_positions=32, c=cache()):
        return lib.bms_rotary_append(PTR, PTR, PTR, dtype, tokens, heads, qs, pair(128, 64), pair(128, 64), PTR, PTR, max_positions, PTR, PTR, PTR,
                                     None if c is None else ctypes.byref(c), None, 0, None)
    for bad in (dict(dtype=5), dict(tokens=-1), dict(heads=0), dict(heads=65536), dict(qs=None), dict(max_positions=0), dict(c=None), dict(c=cache(dim=63)),
                dict(c=cache(dim=0)), dict(c=cache(pages=0)), dict(c=cache(pages=2 ** 31)), dict(c=cache(page_size=0)), dict(c=cache(page_size=65537)),
                dict(c=cache(kv_heads=0)), dict(c=cache(strides=(-1, 64, 64)))):
        assert call(**bad) == INVALID, bad


def test_chunk_attention_refusals(lib):
    def call(dtype=1, tokens=3, heads=4, qs=pair(256, 64), c=cache(), seqs=2, width=4, scale=0.125, window=0, sinks=0):
        return lib.bms_chunk_attention(PTR, dtype, tokens, heads, qs, None if c is None else ctypes.byref(c), PTR, seqs, width, PTR, PTR, scale, window, sinks,
                                       PTR, PTR, PTR, PTR, 1 << 40, 0, None)
    for bad in (dict(dtype=5), dict(tokens=-1), dict(heads=0), dict(heads=3), dict(heads=65536), dict(qs=None), dict(seqs=0), dict(seqs=2 ** 20 + 1),
                dict(width=0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e31), dict(window=-1), dict(sinks=-1), dict(c=None),
                dict(c=cache(kv_heads=3)), dict(c=cache(strides=(2048, -128, 64)))):
        assert call(**bad) == INVALID, bad
    # Positions rounded up to a tile stay in 32 bits; the largest width passes this check (and then fails for want of a device).
    for bad in (dict(c=cache(dim=257)), dict(tokens=2 ** 30), dict(width=2 ** 27), dict(width=(2 ** 31 - 257) // 16 + 1)):
        assert call(**bad) == UNSUPPORTED, bad
    for bad in ((0, -1, 1, 1, 64), (0, 1, 0, 1, 64), (0, 1, 1, 0, 64), (0, 1, 1, 1, 0), (-1, 1, 1, 1, 64), (64, 1, 1, 1, 64)):
        assert lib.bms_attention_workspace_bytes(*bad) == -1, bad


def test_rotary_append_tokens_beyond_a_grid(lib):
    """A block per token: counts that a grid does not hold are refused, not cut to 32 bits."""
    for tokens in (2 ** 31, 2 ** 32 + 5):
        assert lib.bms_rotary_append(PTR, PTR, PTR, 1, tokens, 4, pair(256, 64), pair(128, 64), pair(128, 64), PTR, PTR, 32, PTR, PTR, PTR, ctypes.byref(cache()),
                                     None, 0, None) == UNSUPPORTED


def test_negative_row_strides(lib):
    """They would lead in front of the tensors' memory (the cache's are refused with its shape)."""
    good, bad, c = pair(256, 64), (pair(-256, 64), pair(256, -64)), cache()
    for b in bad:
        for qs, ks, vs in ((b, good, good), (good, b, good), (good, good, b)):
            assert lib.bms_rotary_append(PTR, PTR, PTR, 1, 3, 4, qs, ks, vs, PTR, PTR, 32, PTR, PTR, PTR, ctypes.byref(c), None, 0, None) == INVALID
        assert lib.bms_chunk_attention(PTR, 1, 3, 4, b, ctypes.byref(c), PTR, 2, 4, PTR, PTR, 0.125, 0, 0, PTR, PTR, PTR, PTR, 1 << 40, 0, None) == INVALID


# ---------------------------------------------------------------- Python calls
def fake_cuda():
    """Tensors that claim to be on CUDA: the checks read metadata only."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    return FakeTensorMode()


def test_cpu_tensors_are_never_transferred():
    from bitmask_speculation_b200 import paged
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    x = torch.zeros(2, 4, 8, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="no implicit transfer"):
        paged.PagedCache(x, x)
    with pytest.raises(ValueError, match="no implicit transfer"):
        paged.plan_pages(i, i, i, i[None], i, i[:1], page_size=4, tokens=1)
    with pytest.raises(ValueError, match="no implicit transfer"):
        batched_filtered_sample(torch.zeros(2, 64), None)
    with pytest.raises(ValueError, match="CUDA"):
        batched_filtered_sample(torch.zeros(2, 64), torch.zeros(2, 2, dtype=torch.int32))
    for bad in (torch.zeros(2, 64, dtype=torch.float64), torch.zeros(2, 64, dtype=torch.int32), [[0.0]]):
        with pytest.raises(TypeError):
            batched_filtered_sample(bad, None)


def test_cache_refusals():
    from bitmask_speculation_b200.paged import PagedCache
    with fake_cuda():
        def t(*shape, dtype=torch.bfloat16, device="cuda"):
            return torch.empty(shape, dtype=dtype, device=device)
        ok = t(4, 16, 2, 64)
        assert PagedCache(ok, ok).page_size == 16
        PagedCache(t(4, 2, 16, 64).transpose(1, 2), ok)
        for k, v, error in ((t(4, 16, 128), ok, ValueError), (ok, t(4, 16, 2, 32), ValueError), (ok, t(4, 16, 2, 64, dtype=torch.float16), ValueError),
                            (t(4, 16, 2, 64, dtype=torch.float64), ok, TypeError), (None, ok, TypeError), (t(0, 16, 2, 64), t(0, 16, 2, 64), ValueError),
                            (t(4, 16, 64, 2).transpose(2, 3), ok, ValueError), (t(1, 16, 2, 64).expand(4, 16, 2, 64), ok, ValueError),
                            (t(4, 16, 2, 64, device="cpu"), ok, ValueError)):
            with pytest.raises(error):
                PagedCache(k, v)


def test_plan_refusals():
    from bitmask_speculation_b200.paged import plan_pages
    with fake_cuda():
        def t(*shape, dtype=torch.int32):
            return torch.empty(shape, dtype=dtype, device="cuda")
        good = dict(past_lens=t(3), new_lens=t(3), held=t(3), block_table=t(3, 8), free_pages=t(24), free_count=t(1), page_size=16, tokens=9)
        for change, error in ((dict(past_lens=t(3, dtype=torch.int64)), TypeError), (dict(new_lens=t(4)), ValueError), (dict(held=t(6)[::2]), ValueError),
                              (dict(block_table=t(2, 8)), ValueError), (dict(block_table=t(3, 0)), ValueError), (dict(block_table=t(8, 3).t()), ValueError),
                              (dict(free_pages=t(0)), ValueError), (dict(free_count=t(2)), ValueError), (dict(page_size=0), ValueError),
                              (dict(page_size=16.0), TypeError), (dict(page_size=True), TypeError), (dict(tokens=-1), ValueError), (dict(tokens=2.0), TypeError),
                              (dict(past_lens=t(0), new_lens=t(0), held=t(0), block_table=t(0, 8)), ValueError)):
            with pytest.raises(error):
                plan_pages(**{**good, **change})


def test_append_and_attention_refusals():
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention, rotary_append
    with fake_cuda():
        def t(*shape, dtype=torch.bfloat16):
            return torch.empty(shape, dtype=dtype, device="cuda")
        f32, i32, i64 = torch.float32, torch.int32, torch.int64
        c = PagedCache(t(8, 16, 2, 64), t(8, 16, 2, 64))
        good = dict(q=t(5, 4, 64), k=t(5, 2, 64), v=t(5, 2, 64), cos=t(40, 32, dtype=f32), sin=t(40, 32, dtype=f32), positions=t(5, dtype=i32),
                    slots=t(5, dtype=i64), cache=c)
        for change, error in ((dict(q=t(5, 4, 64, dtype=f32)), TypeError), (dict(q=t(5, 4, 32)), ValueError), (dict(q=t(5, 0, 64)), ValueError),
                              (dict(k=t(4, 2, 64)), ValueError), (dict(v=t(5, 4, 64)), ValueError), (dict(q=t(5, 64, 4).transpose(1, 2)), ValueError),
                              (dict(cos=t(40, 32)), TypeError), (dict(cos=t(40, 64, dtype=f32)), ValueError), (dict(sin=t(32, 40, dtype=f32).t()), ValueError),
                              (dict(cos=t(0, 32, dtype=f32), sin=t(0, 32, dtype=f32)), ValueError), (dict(positions=t(4, dtype=i32)), ValueError),
                              (dict(positions=t(5, dtype=i64)), TypeError), (dict(slots=t(5, dtype=i32)), TypeError), (dict(slots=t(10, dtype=i64)[::2]), ValueError),
                              (dict(status=t(4, dtype=i32)), ValueError), (dict(out=t(5, 4, 64, dtype=f32)), TypeError),
                              (dict(out=t(5, 8, 64)[:, ::2]), ValueError)):
            with pytest.raises(error):
                rotary_append(**{**good, **change})
        good = dict(q=t(5, 4, 64), cache=c, block_table=t(3, 4, dtype=i32), seq_lens=t(3, dtype=i32), query_start=t(4, dtype=i32))
        for change, error in ((dict(q=t(5, 3, 64)), ValueError), (dict(q=t(5, 4, 32)), ValueError), (dict(q=t(4, 64)), ValueError), (dict(block_table=t(2, 4, dtype=i32)), ValueError),
                              (dict(block_table=t(3, 0, dtype=i32)), ValueError), (dict(seq_lens=t(3, dtype=i64)), TypeError), (dict(query_start=t(3, dtype=i32)), ValueError),
                              (dict(window=-1), ValueError), (dict(window=1.5), TypeError), (dict(window=True), TypeError), (dict(sinks=-1), ValueError),
                              (dict(scale="1"), TypeError), (dict(scale=float("nan")), ValueError), (dict(scale=float("inf")), ValueError), (dict(scale=True), TypeError),
                              (dict(out=t(5, 4, 32)), ValueError)):
            with pytest.raises(error):
                chunk_attention(**{**good, **change})


def test_filtered_sample_argument_refusals():
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    with fake_cuda():
        def t(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device="cuda")
        i32 = torch.int32
        logits, mask = t(3, 70), t(3, 3, dtype=i32)
        for change, error in ((dict(mask=t(3, 2, dtype=i32)), ValueError), (dict(mask=t(3, 3)), TypeError), (dict(mask=None, mask_rows=t(3, dtype=i32)), ValueError),
                              (dict(mask_rows=t(2, dtype=i32)), ValueError), (dict(mask_rows=t(3, dtype=torch.int64)), TypeError), (dict(mask=t(0, 3, dtype=i32), mask_rows=t(3, dtype=i32)), ValueError),
                              (dict(logits=t(70, 3).t()), ValueError), (dict(logits=t(3, 0), mask=None), ValueError),
                              (dict(temperature=-1), ValueError), (dict(temperature=float("nan")), ValueError), (dict(temperature="1"), TypeError), (dict(temperature=True), TypeError),
                              (dict(temperature=t(2)), ValueError), (dict(temperature=t(3, dtype=torch.float64)), TypeError), (dict(top_k=-1), ValueError), (dict(top_k=1.0), TypeError),
                              (dict(top_k=t(3)), TypeError), (dict(top_p=0.0), ValueError), (dict(top_p=1.01), ValueError), (dict(min_p=-0.01), ValueError), (dict(min_p=2), ValueError),
                              (dict(min_p=t(6)[::2]), ValueError)):
            with pytest.raises(error):
                batched_filtered_sample(**{**dict(logits=logits, mask=mask), **change})


def test_a_cache_keeps_its_tensors():
    from bitmask_speculation_b200.paged import PagedCache
    with fake_cuda():
        x = torch.empty((4, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
        cache = PagedCache(x, x.clone())
        assert cache.k is x and cache.pages == 4
        for name in ("k", "v", "pages"):
            with pytest.raises(AttributeError):
                setattr(cache, name, x)


def test_a_cache_whose_tensors_moved(monkeypatch):
    """The description follows tensors that were changed in place; ones that no longer match are refused."""
    from bitmask_speculation_b200 import paged
    monkeypatch.setattr(paged, "device_tensor", lambda t, *a, **kw: t)  # tensors on the host: nothing is launched
    k, v = torch.zeros(4, 16, 2, 64), torch.zeros(4, 16, 2, 64)
    cache = paged.PagedCache(k, v)

    def check():
        got = _native.Cache.from_buffer_copy(cache.describe())
        assert (got.k, got.v) == (k.data_ptr(), v.data_ptr())
        assert (got.pages, got.page_size, got.kv_heads, got.dim) == tuple(k.shape)
        assert list(got.k_stride) == list(k.stride()[:3]) and list(got.v_stride) == list(v.stride()[:3])
    check()
    k.data = torch.ones(4, 16, 2, 64)
    check()
    v.set_(torch.ones(4, 2, 16, 64).transpose(1, 2))
    check()
    for t in (k, v):
        t.resize_(9, 16, 2, 64)
    check()
    v.resize_(8, 16, 2, 64)
    with pytest.raises(ValueError, match="share"):
        cache.describe()
    k.resize_(8, 16, 2, 64)
    check()
    k.data = torch.ones(8, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="share"):
        cache.describe()


def test_inputs_that_require_gradients_are_refused(monkeypatch):
    """No result is silently detached; with gradients off the same call passes the checks."""
    from bitmask_speculation_b200 import paged
    reached = []

    class Library:
        def rotary_append(self, *args):
            reached.append("append")

        def chunk_attention(self, *args):
            reached.append("attention")
            return None, None
    monkeypatch.setattr(paged, "load_extension", Library)
    with fake_cuda():
        def t(*shape, dtype=torch.bfloat16):
            return torch.empty(shape, dtype=dtype, device="cuda")
        i32, f32 = torch.int32, torch.float32
        append = dict(q=t(5, 4, 64), k=t(5, 2, 64), v=t(5, 2, 64), cos=t(40, 32, dtype=f32), sin=t(40, 32, dtype=f32), positions=t(5, dtype=i32),
                      slots=t(5, dtype=torch.int64))
        attend = dict(q=t(5, 4, 64), block_table=t(3, 4, dtype=i32), seq_lens=t(3, dtype=i32), query_start=t(4, dtype=i32))
        for call, args, names in ((paged.rotary_append, append, ("q", "k", "v", "cos", "sin", "out", "ck", "cv")), (paged.chunk_attention, attend, ("q", "out", "ck", "cv"))):
            for name in names:
                pages = {"ck": t(8, 16, 2, 64), "cv": t(8, 16, 2, 64)}
                changed = dict(args, **({"out": t(5, 4, 64)} if name == "out" else {}))
                (pages if name in pages else changed)[name].requires_grad_()
                cache = paged.PagedCache(pages["ck"], pages["cv"])
                with pytest.raises(ValueError, match="backward"):
                    call(cache=cache, **changed)
                assert not reached
                with torch.no_grad():
                    call(cache=cache, **changed)
                assert reached.pop() and not reached
                (pages if name in pages else changed)[name].requires_grad_(False)


def test_integers_beyond_64_bits_are_refused():
    """A foreign call would cut them: a window of 2^64 + 5 would be one of 5."""
    from bitmask_speculation_b200.kernels.cuda import batched_filtered_sample
    from bitmask_speculation_b200.paged import PagedCache, chunk_attention, plan_pages
    with fake_cuda():
        def t(*shape, dtype=torch.int32):
            return torch.empty(shape, dtype=dtype, device="cuda")
        bf16 = torch.bfloat16
        cache = PagedCache(t(8, 16, 2, 64, dtype=bf16), t(8, 16, 2, 64, dtype=bf16))
        attend = dict(q=t(5, 4, 64, dtype=bf16), cache=cache, block_table=t(3, 4), seq_lens=t(3), query_start=t(4))
        for change in (dict(window=2 ** 64 + 5), dict(window=2 ** 63), dict(sinks=2 ** 64 + 1), dict(scale=10 ** 400), dict(scale=-10 ** 400)):
            with pytest.raises(ValueError):
                chunk_attention(**{**attend, **change})
        plan = dict(past_lens=t(3), new_lens=t(3), held=t(3), block_table=t(3, 8), free_pages=t(24), free_count=t(1), page_size=16, tokens=9)
        for change in (dict(page_size=2 ** 64 + 16), dict(tokens=2 ** 64 + 9)):
            with pytest.raises(ValueError):
                plan_pages(**{**plan, **change})
        logits = t(3, 70, dtype=torch.float32)
        for change in (dict(top_k=2 ** 63), dict(top_k=10 ** 400), dict(temperature=10 ** 400), dict(top_p=10 ** 400), dict(min_p=float("nan")), dict(top_p=float("-inf"))):
            with pytest.raises(ValueError):
                batched_filtered_sample(logits, None, **change)
