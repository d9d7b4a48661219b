"""Tensor-level selection calls over the sm_100a library.

The functions a caller of the reference imports from kernels/cuda.py:7-69 --
``mask_count``, ``mask_density``, ``masked_argmax``, ``masked_sample`` and
``batched_masked_reduce`` -- with the same arguments, return types and errors,
plus ``batched_masked_sample`` (one uniform per row) and ``batched_filtered_sample``
(temperature, top-k, top-p and min-p per row).  Inputs must already be on
the GPU: nothing here copies, widens or moves a tensor, and a missing library is
an error, never a CPU computation.
"""

from __future__ import annotations

from dataclasses import dataclass

from ._extension import load_extension
from ._validation import (batched_selection_inputs, filter_value, index_tensor, mask_input, selection_inputs,
                          temperature_input, uniforms_input)

_MESSAGES = {
    1: "mask has no valid token",
    2: "logits contain NaN",
    3: "uniform must be finite and in [0, 1)",
    4: "valid logits have no finite probability mass",
    5: "positive infinity is unsupported for stochastic sampling",
    7: "device wait timed out",
}


def mask_count(mask, vocab_size: int):
    """Valid tokens of one packed mask row, as a new 0-d int64 tensor on the mask's device.
    Enqueued on the current stream; the host does not wait."""
    vocab_size = mask_input(mask, vocab_size)
    return load_extension().mask_count(mask, vocab_size)


def mask_density(mask, vocab_size: int):
    """``mask_count / vocab_size`` as a 0-d float64 tensor on the device (no host wait)."""
    import torch
    return mask_count(mask, vocab_size).to(torch.float64) / vocab_size


def _checked_selection(result):
    output, status = result[0], result[-1]
    code = status.item()  # the one device->host read of the call
    if code in _MESSAGES:
        raise ValueError(_MESSAGES[code])
    if code != 0:
        raise RuntimeError(f"unknown native selection status: {code}")
    return output


def masked_argmax(logits, mask):
    """Highest-scoring allowed token of one row (ties: smallest ID) as a new 0-d int64 tensor.
    Reads the status back to the host once, raising ValueError for NaN or an empty mask."""
    selection_inputs(logits, mask)
    return _checked_selection(load_extension().masked_argmax(logits, mask))


def masked_sample(logits, mask, *, temperature: float = 1.0, generator=None):
    """Draw one allowed token from softmax(logits / temperature) by inverse CDF.

    ``temperature == 0`` is ``masked_argmax``.  Otherwise one float64 uniform is
    drawn on the logits' device from ``generator`` (the device default if None),
    after the library is loaded so that a load failure leaves the generator
    untouched.  The status is read back once (ValueError on a data error).  One
    row, one draw: speculative acceptance lives elsewhere.
    """
    import torch
    temperature = temperature_input(temperature)
    selection_inputs(logits, mask)
    if temperature == 0:
        return masked_argmax(logits, mask)
    native = load_extension()  # before the draw: a failed load leaves the generator as it was
    uniform = torch.rand((), dtype=torch.float64, device=logits.device, generator=generator)
    return _checked_selection(native.masked_sample(logits, mask, temperature, uniform))


@dataclass(frozen=True, slots=True)
class BatchedMaskedReduction:
    """Per-row results of a batched call: token (-1 on error), valid count, status code.
    ``check()`` reads the statuses back once and raises ValueError listing failed rows."""

    token_ids: object
    valid_counts: object
    status: object

    def check(self) -> "BatchedMaskedReduction":
        codes = self.status.tolist()  # reads every row's status back in one transfer
        errors = [(row, code) for row, code in enumerate(codes) if code]
        if errors:
            raise ValueError(f"invalid reduction rows (row, status): {errors}")
        return self


def batched_masked_reduce(logits, mask):
    """Masked argmax, valid-token count and status of every row of a [B, V] batch under its
    [B, ceil(V/32)] masks, as new [B] tensors on the device.  The whole batch is one selection
    launch; the host does not wait."""
    batched_selection_inputs(logits, mask)
    tokens, counts, status = load_extension().masked_reduce_batch(logits, mask)
    return BatchedMaskedReduction(tokens, counts, status)


def batched_masked_sample(logits, mask, *, temperature: float, uniforms=None, generator=None):
    """Sample every row of a batch; one float64 uniform per row (drawn if not given).

    Returns a ``BatchedMaskedReduction`` (token, valid count, status per row).
    """
    import torch
    temperature = temperature_input(temperature)
    batch, _ = batched_selection_inputs(logits, mask)
    native = load_extension()
    if temperature == 0:
        tokens, counts, status = native.masked_reduce_batch(logits, mask)
        return BatchedMaskedReduction(tokens, counts, status)
    if uniforms is None:
        uniforms = torch.rand(batch, dtype=torch.float64, device=logits.device, generator=generator)
    uniforms_input(uniforms, batch, logits.device)
    tokens, counts, status = native.masked_sample_batch(logits, mask, temperature, uniforms)
    return BatchedMaskedReduction(tokens, counts, status)


@dataclass(frozen=True, slots=True)
class FilteredSample:
    """Per-row results of ``batched_filtered_sample``: token (-1 on error), number of tokens the
    filters kept (0 on error), status code.  ``check()`` reads the statuses back once and raises
    ValueError listing failed rows."""

    token_ids: object
    kept_counts: object
    status: object

    def check(self) -> "FilteredSample":
        errors = [(row, code) for row, code in enumerate(self.status.tolist()) if code]
        if errors:
            raise ValueError(f"invalid filtered rows (row, status): {errors}")
        return self


def batched_filtered_sample(logits, mask, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, uniforms=None,
                            generator=None, mask_rows=None):
    """Sample every row of a [B, V] batch from its filtered masked softmax; one float64 uniform per row
    (drawn if not given).

    A row's valid finite tokens are ordered by (logit descending, token ascending) and weigh
    exp((x - max) / temperature).  Kept is the shortest of three prefixes of that order: the first
    ``top_k`` tokens (0: off); of their mass, the tokens whose preceding mass is below ``top_p`` times it
    (1: off); the tokens weighing at least ``min_p`` (0: off).  The result is the lowest kept token
    whose running mass in token order exceeds the uniform times the kept mass.  ``temperature`` 0 is
    the masked argmax.  Each parameter is a number or a [B] tensor on the device (float32; int32 for
    ``top_k``), mixed as needed; a row whose value is out of range fails with status 10.

    ``mask``: [B, ceil(V / 32)] int32 rows, or None (every token allowed); with ``mask_rows`` (int32
    [B] on the device) ``mask`` is a table [R, ceil(V / 32)] and row r uses ``mask[mask_rows[r]]`` (status 8
    for an index outside it).  The other statuses are the sampler's.  Weights and sums are float64, in
    an order that the call's shapes fix: the same call gives the same results.  A row in a batch of another size may be
    summed in another order; it could come out differently only where its uniform or a filter's limit lies within float64
    rounding of a boundary.  No host synchronization.
    """
    import torch
    if mask is None:
        if mask_rows is not None:
            raise ValueError("mask_rows needs a mask table")
        if not isinstance(logits, torch.Tensor) or logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError("logits must be a float32, bfloat16 or float16 tensor")
        if logits.layout != torch.strided or logits.ndim != 2 or not logits.is_contiguous() or logits.shape[1] == 0:
            raise ValueError("logits must be a contiguous [batch, vocab] tensor")
        if logits.device.type != "cuda":
            raise ValueError("logits must be on CUDA; no implicit transfer")
        batch = logits.shape[0]
    elif mask_rows is None:
        batch, _ = batched_selection_inputs(logits, mask)
    else:
        if not isinstance(mask, torch.Tensor) or mask.ndim != 2 or mask.shape[0] == 0:
            raise ValueError("mask must be a table [R, ceil(vocab_size / 32)]")
        batched_selection_inputs(logits[:0], mask[:0])
        batch = logits.shape[0]
        if not logits.is_contiguous() or not mask.is_contiguous():
            raise ValueError("batch inputs must be contiguous two-dimensional strided tensors")
        if index_tensor(mask_rows, "mask_rows", ndim=1, device=logits.device).shape[0] != batch:
            raise ValueError("mask_rows must have one index per row")
    dev = logits.device
    temperature = filter_value(temperature, "temperature", batch, dev, low=0.0, high=1.7976931348623157e308)
    top_k = filter_value(top_k, "top_k", batch, dev, low=0, high=2 ** 63 - 1, integer=True)
    top_p = filter_value(top_p, "top_p", batch, dev, low=0.0, high=1.0, low_open=True)
    min_p = filter_value(min_p, "min_p", batch, dev, low=0.0, high=1.0)
    native = load_extension()
    if uniforms is None:
        uniforms = torch.rand(batch, dtype=torch.float64, device=dev, generator=generator)
    uniforms_input(uniforms, batch, dev)
    return FilteredSample(*native.filtered_sample_batch(logits, mask, mask_rows, temperature, top_k, top_p, min_p, uniforms))
