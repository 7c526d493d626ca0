"""The paged KV cache in microscaled 4-bit floating point.

A row (one token of one KV head) of K or V is ``head_dim/2`` bytes of e2m1
codes, two to a byte with the lower dim in the low nibble, and 4 scale bytes of
which the first ``head_dim/32`` are used: byte j is the power of two
``2^(byte - 127)`` of dims [32j, 32j + 32), 255 meaning NaN. That is 4.25 bits
a value at head_dim 128 against 16, laid out as the fp16 cache is::

    k_cache, v_cache    [num_pages, page_size, Hkv, head_dim / 2]  uint8
    k_scales, v_scales  [num_pages, page_size, Hkv, 4]             uint8

The reference has no counterpart.
"""

from __future__ import annotations

import math

import torch

from . import _lib, kernel_cuda_v4
from .decode_weights import _new_tokens
from .kernel_cuda_v4 import _check_own_pages, _check_positions, _raise_flags_of, read_error_flags

_OPS = _lib.ops()
FP4_HEAD_DIMS = (32, 64, 128)


def paged_kv_cache_fp4(num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, device="cuda"):
    """A new cache of zeros: (k_cache, k_scales, v_cache, v_scales)."""
    assert head_dim in FP4_HEAD_DIMS, f"head_dim must be one of {FP4_HEAD_DIMS}"
    rows = (num_pages, page_size, num_kv_heads)
    new = lambda n: torch.zeros((*rows, n), dtype=torch.uint8, device=device)  # noqa: E731
    return new(head_dim // 2), new(4), new(head_dim // 2), new(4)


def paged_kv_append_fp4(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, k_scales: torch.Tensor,
                        v_cache: torch.Tensor, v_scales: torch.Tensor, block_table: torch.Tensor,
                        positions: torch.Tensor, seq_ids: torch.Tensor | None = None) -> None:
    """Quantise new tokens and write them into the 4-bit cache in place.

    Row t of k_new / v_new [tokens, Hkv, D] fp16 becomes token positions[t] of
    sequence seq_ids[t] (None: of sequence t, one token of each sequence at
    most), so one call takes a decoding step or whole prompts; positions[t] < 0
    skips t. Per block of 32 dims the scale is the power of two that puts the
    largest magnitude into [4, 8), at least 2^-24, and the codes are rounded to
    nearest even and saturate at 6; a block with an Inf or NaN becomes NaN. A
    call must not name the same (sequence, position) twice."""
    assert k_new.is_cuda and k_cache.is_cuda, "pad_b200 requires CUDA tensors"
    assert k_new.dtype == torch.float16 and v_new.dtype == torch.float16, "pad_b200 expects fp16 k_new/v_new"
    assert k_new.dim() == 3 and k_new.shape[2] in FP4_HEAD_DIMS, f"head_dim must be one of {FP4_HEAD_DIMS}"
    assert seq_ids is not None or k_new.shape[0] <= block_table.shape[0], "more tokens than sequences need seq_ids"
    if kernel_cuda_v4._CHECK_VALUES:
        read_error_flags(k_cache.device)
    _OPS.kv_append_fp4(k_new, v_new, k_cache, k_scales, v_cache, v_scales, block_table, positions, seq_ids)
    if kernel_cuda_v4._CHECK_VALUES:
        _raise_flags_of(k_cache.device)


def paged_kv_read_fp4(k_cache: torch.Tensor, k_scales: torch.Tensor, v_cache: torch.Tensor, v_scales: torch.Tensor,
                      block_table: torch.Tensor, positions: torch.Tensor, seq_ids: torch.Tensor | None = None):
    """The fp16 values (k, v) [tokens, Hkv, D] that the 4-bit cache holds for
    token positions[t] of sequence seq_ids[t] (None: of sequence t) -- what a
    later chunk of a prompt attends to. Exact for rows written by
    paged_kv_append_fp4; positions[t] < 0 reads as zeros."""
    assert k_cache.is_cuda, "pad_b200 requires CUDA tensors"
    assert 2 * k_cache.shape[3] in FP4_HEAD_DIMS, f"head_dim must be one of {FP4_HEAD_DIMS}"
    assert seq_ids is not None or positions.shape[0] <= block_table.shape[0], "more tokens than sequences need seq_ids"
    if kernel_cuda_v4._CHECK_VALUES:
        read_error_flags(k_cache.device)
    got = _OPS.kv_read_fp4(k_cache, k_scales, v_cache, v_scales, block_table, positions, seq_ids)
    if kernel_cuda_v4._CHECK_VALUES:
        _raise_flags_of(k_cache.device)
    return got


def paged_attention_decode_fp4(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    k_scales: torch.Tensor,
    v_cache: torch.Tensor,
    v_scales: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    num_splits: int | None = None,
    scale: float | None = None,
    *,
    weights: torch.Tensor | None = None,
    num_new: int | torch.Tensor = 1,
    slot_positions: torch.Tensor | None = None,
    total_lens: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Decode attention over the 4-bit cache: paged_attention_decode_cuda_v4 with
    K and V what their codes and scales stand for.

    q [B, Hq, D] fp16 -> out [B, Hq, D] fp16; head_dim 32, 64 or 128, up to 16
    query heads per KV head. V's scales lie in 2^-24 .. 2^13 as the append
    writes them: a smaller one counts as 0, a larger one (not NaN) is flagged
    (an error with PAD_B200_CHECK=1) and its sequence's output undefined.
    weights, num_new, slot_positions and total_lens are those of
    paged_attention_decode_weights (weights=None: not tracked)."""
    assert q.is_cuda and k_cache.is_cuda and v_cache.is_cuda, "pad_b200 requires CUDA tensors"
    assert q.dtype == torch.float16 and q.dim() == 3, "pad_b200 expects fp16 q [B, Hq, D]"
    _, num_q_heads, head_dim = q.shape
    assert head_dim in FP4_HEAD_DIMS, f"head_dim must be one of {FP4_HEAD_DIMS}"
    assert num_q_heads % k_cache.shape[2] == 0, "num_q_heads must be divisible by num_kv_heads (GQA)"
    assert num_splits is None or num_splits >= 1, "num_splits must be >= 1"
    new, num_new_of = num_new, None
    if type(num_new) is not int:
        num_new, num_new_of = _new_tokens(num_new)
    assert num_new >= 0, "num_new must be >= 0"
    assert weights is not None or slot_positions is None, "slot_positions go with weights"
    assert slot_positions is not None or total_lens is None, "total_lens goes with slot_positions"
    if slot_positions is not None and total_lens is None:
        total_lens = seq_lens
        if kernel_cuda_v4._CHECK_VALUES:
            _check_positions(slot_positions, total_lens, block_table, seq_lens, new)
    if kernel_cuda_v4._CHECK_VALUES:
        read_error_flags(q.device)
        if weights is not None:
            _check_own_pages(block_table, seq_lens, k_cache.shape[1])
    out = _OPS.decode_fp4(q, k_cache, k_scales, v_cache, v_scales, block_table, seq_lens,
                          0 if num_splits is None else int(num_splits),
                          float(scale) if scale is not None else 1.0 / math.sqrt(head_dim), out, weights, num_new,
                          slot_positions, total_lens, num_new_of)
    if kernel_cuda_v4._CHECK_VALUES:
        _raise_flags_of(q.device)
    return out
