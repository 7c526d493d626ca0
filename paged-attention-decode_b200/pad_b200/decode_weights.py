"""Decode that also accumulates each cached token's attention weight -- what an
eviction (pad_b200.evict) decides by. The reference has no counterpart."""

from __future__ import annotations

import math

import torch

from . import _lib, kernel_cuda_v4
from .kernel_cuda_v4 import _SUPPORTED_HEAD_DIMS, _check_own_pages, _check_positions, _raise_flags_of, read_error_flags

_OPS = _lib.ops()


def _new_tokens(num_new: int | torch.Tensor) -> tuple[int, torch.Tensor | None]:
    """num_new as the operators take it, unless it is an int: a number, or a tensor with one of each sequence."""
    if isinstance(num_new, torch.Tensor):
        return 0, num_new
    return int(num_new), None


def paged_attention_decode_weights(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    weights: torch.Tensor,
    num_new: int | torch.Tensor = 1,
    num_splits: int | None = None,
    scale: float | None = None,
    *,
    slot_positions: torch.Tensor | None = None,
    total_lens: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """paged_attention_decode_cuda_v4, and ``weights`` updated in place.

    weights [num_pages, Hkv, page_size] fp32 gains, for every cached token and
    KV head, the token's softmax probability summed over the KV head's query
    heads. The num_new last tokens of each sequence are new: their weight is
    set, not added to, so a page's slots need no clearing before they are used
    (num_new = 0 only adds). num_new is one number for every sequence or an
    integer tensor [B], one of each: 1 for those that decode, the length of its
    prompt for one that has just joined them (below 0 counts as 0).
    slot_positions [num_pages, Hkv, page_size] int32, if given, gets the new
    tokens' positions, counted from total_lens [B] (the tokens each sequence has
    seen; None: seq_lens, which is right before a first eviction only, and refused
    later with PAD_B200_CHECK=1: the new tokens would get positions that older
    ones have). Sequences must not share pages (their weights would lose
    additions, other ones from run to run; refused with PAD_B200_CHECK=1)."""
    assert q.is_cuda and k_cache.is_cuda and v_cache.is_cuda, "pad_b200 requires CUDA tensors"
    assert q.dtype == torch.float16 and k_cache.dtype == torch.float16 and v_cache.dtype == torch.float16, (
        "pad_b200 expects fp16 q/k_cache/v_cache"
    )
    # (shapes that only have to agree are checked by the operator)
    assert q.dim() == 3 and k_cache.dim() == 4, "q must be [B, Hq, D] and k_cache [num_pages, page_size, Hkv, D]"
    _, num_q_heads, head_dim = q.shape
    assert num_q_heads % k_cache.shape[2] == 0, "num_q_heads must be divisible by num_kv_heads (GQA)"
    assert head_dim in _SUPPORTED_HEAD_DIMS, f"head_dim must be one of {_SUPPORTED_HEAD_DIMS}"
    assert num_splits is None or num_splits >= 1, "num_splits must be >= 1"
    new, num_new_of = num_new, None
    if type(num_new) is not int:
        num_new, num_new_of = _new_tokens(num_new)
    assert num_new >= 0, "num_new must be >= 0"
    assert slot_positions is not None or total_lens is None, "total_lens goes with slot_positions"
    if slot_positions is not None and total_lens is None:
        total_lens = seq_lens
        if kernel_cuda_v4._CHECK_VALUES:
            _check_positions(slot_positions, total_lens, block_table, seq_lens, new)
    if kernel_cuda_v4._CHECK_VALUES:
        read_error_flags(q.device)
        _check_own_pages(block_table, seq_lens, k_cache.shape[1])
    out = _OPS.decode_weights(q, k_cache, v_cache, block_table, seq_lens, 0 if num_splits is None else int(num_splits),
                              float(scale) if scale is not None else 1.0 / math.sqrt(head_dim), out, weights,
                              num_new, slot_positions, total_lens, num_new_of)
    if kernel_cuda_v4._CHECK_VALUES:
        _raise_flags_of(q.device)
    return out
