"""Paged key/value cache of a serving round: page planning, rotary append, chunk attention.

The reference forwards its models through Transformers (models/transformers.py:147-201) and has no cache of its
own; these operators have no reference counterpart.  A round of speculative decoding uses them in this order:

* ``plan_pages`` brings every sequence's block table to the round's lengths on the device (drafts that were
  rejected shrink, windows and prompts grow, finished requests give their pages back) and gives the
  new tokens' positions and cache slots;
* per layer, ``rotary_append`` rotates the new queries and keys and writes keys and values into the
  pages, and ``chunk_attention`` attends with the new rows (one token, a K + 1 window or a prompt
  chunk per sequence, mixed in one call) over everything the block tables reach;
* the logits go to ``verify_batch`` or ``batched_filtered_sample``.

Nothing synchronises with the host, every call runs on the current stream of its tensors' device, and
each can be captured into a CUDA graph.  Inputs must already be on the GPU; a missing library is an
error, never a CPU computation.  There is no backward pass: inputs that require gradients are refused unless gradients
are off.
"""

from __future__ import annotations

import math
import struct
import sys
from dataclasses import dataclass

from .kernels._extension import load_extension
from .kernels._validation import device_tensor, index_tensor


_INT64_MAX = 2 ** 63 - 1  # the C library's integers: ctypes would cut larger ones without a word
_PACK = struct.Struct("2P10q").pack  # bms_paged_cache: k, v, shape, k's strides, v's strides


def _check_pages(k, v) -> None:
    device_tensor(k, "k", ndim=4, floating=True)
    device_tensor(v, "v", ndim=4, floating=True)
    if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
        raise ValueError("k and v must share shape, dtype and device")
    if k.numel() == 0:
        raise ValueError("the cache must not be empty")
    if k.stride(3) != 1 or v.stride(3) != 1:
        raise ValueError("the head dimension must be contiguous")
    for t in (k, v):
        if any(n > 1 and s <= 0 for n, s in zip(t.shape, t.stride())):
            raise ValueError("cache strides must be positive")


def _form(k, v):
    return k.shape, k.stride(), v.shape, v.stride(), k.dtype, v.dtype


class PagedCache:
    """Keys and values in pages: ``k`` and ``v`` [pages, page_size, kv_heads, dim], float32, bfloat16 or
    float16, on one CUDA device, ``dim`` contiguous, any other strides (a [pages, kv_heads, page_size,
    dim] layout is passed as its transposed view).  Slot j of page p is slot p * page_size + j.  A cache keeps
    its tensors: other ones make another cache.  Every call reads the tensors as they are: one whose memory, shape or
    strides were changed in place (``resize_``, ``set_``, ``.data``) is checked again."""

    __slots__ = ("_k", "_v", "_form")

    def __init__(self, k, v):
        _check_pages(k, v)
        self._k, self._v = k, v
        self._form = _form(k, v)

    @classmethod
    def allocate(cls, pages: int, page_size: int, kv_heads: int, dim: int, *, dtype=None, device="cuda") -> "PagedCache":
        """A zeroed cache of ``pages`` pages (bfloat16 unless given)."""
        import torch
        shape = (pages, page_size, kv_heads, dim)
        dtype = torch.bfloat16 if dtype is None else dtype
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    def describe(self):
        """The C library's ``bms_paged_cache`` of the tensors as they are now."""
        k, v = self._k, self._v
        form = _form(k, v)
        if form != self._form:
            _check_pages(k, v)
            self._form = form
        return _PACK(k.data_ptr(), v.data_ptr(), *form[0], *form[1][:3], *form[3][:3])

    @property
    def k(self):
        return self._k

    @property
    def v(self):
        return self._v

    @property
    def pages(self) -> int:
        return self.k.shape[0]

    @property
    def page_size(self) -> int:
        return self.k.shape[1]


@dataclass(frozen=True, slots=True)
class PagePlan:
    """Device tensors of one step: ``query_start`` [S + 1], ``seq_lens`` [S] (with the new tokens), per
    packed token ``positions`` int32 and ``slots`` int64 [tokens] (-1 behind the last sequence and for failed
    ones), the pages each sequence now holds, the new free count [1], and a status per sequence (0; 6:
    lengths that do not fit; 9: the pool ran out)."""

    query_start: object
    seq_lens: object
    positions: object
    slots: object
    held: object
    free_count: object
    status: object

    def check(self) -> "PagePlan":
        """Reads the statuses back once and raises ``ValueError`` listing failed sequences."""
        _raise_failed(self.status, "invalid plan sequences")
        return self


@dataclass(frozen=True, slots=True)
class ChunkAttention:
    """``out`` [tokens, heads, dim], ``lse`` float32 [tokens, heads] (natural log of the sum of
    exponentials) and a status per sequence (0; 6: lengths that do not fit, or rows that another sequence
    claims too; 7: a wait inside the kernel gave up; 11: a page outside the cache; the rows of a failed sequence that
    belong to no other one are 0 with lse -inf)."""

    out: object
    lse: object
    status: object

    def check(self) -> "ChunkAttention":
        """Reads the statuses back once and raises ``ValueError`` listing failed sequences."""
        _raise_failed(self.status, "invalid attention sequences")
        return self


def _raise_failed(status, what: str) -> None:
    errors = [(s, code) for s, code in enumerate(status.tolist()) if code]
    if errors:
        raise ValueError(f"{what} (sequence, status): {errors}")


def plan_pages(past_lens, new_lens, held, block_table, free_pages, free_count, *, page_size: int, tokens: int) -> PagePlan:
    """Block tables, positions and slots of one step, from the requests' lengths.

    Sequence s keeps ``past_lens[s]`` tokens and appends ``new_lens[s]``; it holds the first ``held[s]``
    entries of ``block_table`` [S, width] and ends with exactly ceil((past + new) / page_size) of them.
    Surplus pages go back to the pool first (a finished request: past = new = 0), lacking ones are popped from
    the stack ``free_pages`` [pages] of which ``free_count`` [1] entries are free.  All int32.
    ``tokens`` is the packed step's row count (the host knows it); rows behind the last sequence get
    position and slot -1.  ``block_table`` and ``free_pages`` are updated in place and stay consistent
    with the returned ``held`` and ``free_count``; a failed sequence keeps its pages and gets
    ``seq_lens`` 0.  At most 8,192 sequences.
    """
    seqs = index_tensor(past_lens, "past_lens", ndim=1).shape[0]
    dev = past_lens.device
    for t, name in ((new_lens, "new_lens"), (held, "held")):
        if index_tensor(t, name, ndim=1, device=dev).shape[0] != seqs:
            raise ValueError(f"{name} must be an int32 [S] tensor")
    if index_tensor(block_table, "block_table", ndim=2, device=dev).shape[0] != seqs:
        raise ValueError("block_table must be an int32 [S, width] tensor")
    index_tensor(free_pages, "free_pages", ndim=1, device=dev)
    if index_tensor(free_count, "free_count", ndim=1, device=dev).shape[0] != 1:
        raise ValueError("free_count must be an int32 [1] tensor")
    _positive_int(page_size, "page_size")
    if isinstance(tokens, bool) or not isinstance(tokens, int):
        raise TypeError("tokens must be an integer")
    if not 0 <= tokens <= _INT64_MAX:
        raise ValueError("tokens must be in [0, 2^63)")
    if seqs == 0 or block_table.shape[1] == 0 or free_pages.shape[0] == 0:
        raise ValueError("the plan needs sequences, table entries and pages")
    return PagePlan(*load_extension().page_plan(past_lens, new_lens, held, block_table, free_pages, free_count, page_size, tokens))


def rotary_append(q, k, v, cos, sin, positions, slots, cache: PagedCache, *, out=None, status=None):
    """Rotate a step's queries and keys, write keys and values into the cache, return the queries.

    ``q`` [N, heads, dim], ``k`` and ``v`` [N, kv_heads, dim] of the cache's dtype (views of one
    projection's output are fine: the last dimension is contiguous, other strides are free); ``cos`` and ``sin``
    float32 [max_positions, dim / 2]; ``positions`` int32 and ``slots`` int64 [N], as ``plan_pages``
    gives them.  Element i and i + dim / 2 of a head turn together; sums are float32, rounded once.  A
    token with slot -1 writes no key or value; one with position -1 nothing, its row of the result is
    left as it was (unspecified when ``out`` is not given).  ``out``: a contiguous tensor shaped like ``q`` for
    the result (a contiguous ``q`` itself may be given; it overlaps nothing else).  ``status``: an int32 [N] tensor for a code per token (0; 11: a slot outside the cache;
    12: a position outside the tables; such tokens write nothing).
    """
    import torch
    pages = cache.k
    dtype, dev = pages.dtype, pages.device
    device_tensor(q, "q", ndim=3, dtype=dtype, device=dev)
    device_tensor(k, "k", ndim=3, dtype=dtype, device=dev)
    device_tensor(v, "v", ndim=3, dtype=dtype, device=dev)
    n, heads, dim = q.shape
    if dim % 2 or dim != pages.shape[3] or heads == 0:
        raise ValueError("q's head dimension must be even and equal the cache's")
    if k.shape != v.shape or tuple(k.shape) != (n, pages.shape[2], dim):
        raise ValueError("k and v must be [N, kv_heads, dim] tensors")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _row_strides(t, name)
    device_tensor(cos, "cos", ndim=2, dtype=torch.float32, device=dev)
    device_tensor(sin, "sin", ndim=2, dtype=torch.float32, device=dev)
    if cos.shape != sin.shape or cos.shape[1] * 2 != dim or cos.shape[0] == 0 or not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("cos and sin must be contiguous [max_positions, dim / 2] tensors")
    index_tensor(positions, "positions", ndim=1, device=dev)
    index_tensor(slots, "slots", ndim=1, device=dev, dtype=torch.int64)
    if positions.shape[0] != n or slots.shape[0] != n:
        raise ValueError("positions and slots must have one entry per token")
    if status is not None and index_tensor(status, "status", ndim=1, device=dev).shape[0] != n:
        raise ValueError("status must be an int32 [N] tensor")
    if torch.is_grad_enabled():
        _no_gradients(q, k, v, cos, sin, out, pages, cache.v)
    if out is None:
        out = torch.empty((n, heads, dim), dtype=dtype, device=dev)
    else:
        _output(out, q, "out")
    load_extension().rotary_append(q, k, v, cos, sin, positions, slots, out, cache, status)
    return out


def chunk_attention(q, cache: PagedCache, block_table, seq_lens, query_start, *, scale: float | None = None,
                    window: int = 0, sinks: int = 0, out=None) -> ChunkAttention:
    """Attention of each sequence's new rows over its pages, which already hold the new keys and values.

    ``q`` [N, heads, dim] (dim at most 256, heads a multiple of the cache's kv_heads, strides as for
    ``rotary_append``); sequence s owns rows [query_start[s], query_start[s + 1]) and has ``seq_lens[s]``
    tokens in the pages of ``block_table`` row s, its rows the last of them.  Row i at position p sees the
    keys j <= p; with ``window`` > 0 only those with p - j < window, and the first ``sinks`` ones.
    ``scale`` is 1 / sqrt(dim) unless given.  Keys that a row does not see never reach it, whatever
    they hold.  ``block_table`` int32 [S, width], ``seq_lens`` int32 [S], ``query_start`` int32
    [S + 1].  Rows behind the last sequence are left as they were (unspecified when ``out`` is not given).
    A row whose visible scores are all -inf is NaN with lse -inf; one that sees a score of +inf or NaN is NaN with
    lse NaN.  ``out`` must not overlap the inputs.

    Tensor cores take 16-bit types of dim 64 or 128 in pages that divide 128 slots or are divided by them (8 slots at
    least), with bases and strides on 16-byte boundaries and no broadcast; every other call goes row by row, which is
    meant for small ones (long float32 caches and prompts take longer than elementary operations do).
    """
    import torch
    pages = cache.k
    dtype, dev = pages.dtype, pages.device
    device_tensor(q, "q", ndim=3, dtype=dtype, device=dev)
    n, heads, dim = q.shape
    kv_heads = pages.shape[2]
    if dim != pages.shape[3] or dim > 256:
        raise ValueError("q's head dimension must equal the cache's and be at most 256")
    if heads == 0 or heads % kv_heads:
        raise ValueError("heads must be a multiple of the cache's kv_heads")
    _row_strides(q, "q")
    seqs = index_tensor(seq_lens, "seq_lens", ndim=1, device=dev).shape[0]
    if index_tensor(block_table, "block_table", ndim=2, device=dev).shape[0] != seqs:
        raise ValueError("block_table must be an int32 [S, width] tensor")
    if index_tensor(query_start, "query_start", ndim=1, device=dev).shape[0] != seqs + 1:
        raise ValueError("query_start must be an int32 [S + 1] tensor")
    if seqs == 0 or block_table.shape[1] == 0:
        raise ValueError("the call needs sequences and table entries")
    for value, name in ((window, "window"), (sinks, "sinks")):
        if isinstance(value, bool) or not isinstance(value, int):
            raise TypeError(f"{name} must be an integer")
        if not 0 <= value <= _INT64_MAX:
            raise ValueError(f"{name} must be in [0, 2^63)")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    elif isinstance(scale, bool) or not isinstance(scale, (int, float)):
        raise TypeError("scale must be numeric")
    elif not abs(scale) <= sys.float_info.max:  # NaN, infinities and integers that no float holds
        raise ValueError("scale must be finite")
    if torch.is_grad_enabled():
        _no_gradients(q, out, pages, cache.v)
    if out is None:
        out = torch.empty((n, heads, dim), dtype=dtype, device=dev)
    else:
        _output(out, q, "out")
    lse, status = load_extension().chunk_attention(q, cache, block_table, seq_lens, query_start, float(scale), window, sinks, out)
    return ChunkAttention(out, lse, status)


def _positive_int(value, name: str) -> None:
    if isinstance(value, bool) or not isinstance(value, int):
        raise TypeError(f"{name} must be an integer")
    if not 0 < value <= _INT64_MAX:
        raise ValueError(f"{name} must be positive and below 2^63")


def _no_gradients(*tensors) -> None:
    if any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("the cache operators have no backward pass: detach the inputs or call them under torch.no_grad()")


def _row_strides(t, name: str) -> None:
    if t.stride(2) != 1 and t.shape[2] > 1 and t.numel():
        raise ValueError(f"{name}'s last dimension must be contiguous")


def _output(out, like, name: str) -> None:
    device_tensor(out, name, ndim=3, dtype=like.dtype, device=like.device)
    if out.shape != like.shape or not out.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of q's shape")


__all__ = ["PagedCache", "PagePlan", "ChunkAttention", "plan_pages", "rotary_append", "chunk_attention"]
