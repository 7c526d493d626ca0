"""Eviction from a paged cache by accumulated attention weight.

Beside the cache live ``weights`` (fp32) and, if recent tokens are to be kept
whatever they weigh, ``slot_positions`` (int32), both [num_pages, Hkv,
page_size] and addressed through the cache's block table: what each slot's
token has received so far (the decode with weights adds to it) and the token's
position in its sequence. Every KV head keeps its own tokens. The reference has
no counterpart.
"""

from __future__ import annotations

from typing import Sequence

import torch

from . import _lib, kernel_cuda_v4
from .kernel_cuda_v4 import _check_own_pages, _check_positions, _raise_flags_of, read_error_flags

_OPS = _lib.ops()


def paged_kv_evict_plan(weights: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, budget: int,
                        recent: int = 0, *, slot_positions: torch.Tensor | None = None,
                        total_lens: torch.Tensor | None = None):
    """Which slots to keep, as the moves that make them the first ``budget``.

    For every sequence with seq_lens[b] > budget and every KV head the slots
    kept are first those whose slot_positions are at least total_lens[b] -
    recent (total_lens [B]: tokens the sequence has seen; None: seq_lens, which
    is right before a first eviction only, and refused later with
    PAD_B200_CHECK=1: too many tokens would count as recent), then the heaviest
    (NaN above all), ties to the lower slot. Returns (src, dst, counts,
    new_lens): move i < counts[b, h] copies slot src[b, h, i] to dst[b, h, i]
    (both ascending, -1 behind the last), and new_lens = min(seq_lens, budget).
    Slots keep their place unless they lie at or above the budget, so their
    order says nothing about age afterwards; attention does not depend on it.
    Sequences must not share pages: moving one's rows would overwrite the
    other's (refused with PAD_B200_CHECK=1)."""
    assert weights.is_cuda, "pad_b200 requires CUDA tensors"
    assert weights.dtype == torch.float32 and weights.dim() == 3, "weights must be fp32 [num_pages, Hkv, page_size]"
    assert budget >= 1, "budget must be >= 1"
    assert 0 <= recent <= budget, "recent must lie in [0, budget]"
    assert recent == 0 or slot_positions is not None, "recent needs slot_positions"
    if slot_positions is not None and total_lens is None:
        total_lens = seq_lens
    if kernel_cuda_v4._CHECK_VALUES:
        read_error_flags(weights.device)
        _check_own_pages(block_table, seq_lens, weights.shape[2])
        if recent > 0:
            _check_positions(slot_positions, total_lens, block_table, seq_lens)
    got = _OPS.kv_evict_plan(weights, block_table, seq_lens, budget, recent, slot_positions,
                             total_lens if slot_positions is not None else None)
    if kernel_cuda_v4._CHECK_VALUES:
        _raise_flags_of(weights.device)
    return got


def _check_moves(cache: torch.Tensor, block_table: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
                 counts: torch.Tensor) -> None:
    """Refuse moves whose target is a source or the target of another."""
    if (cache.dim() != 4 or src.dim() != 3 or dst.shape != src.shape or counts.shape != src.shape[:2] or
            block_table.dim() != 2 or block_table.shape[0] != src.shape[0]):
        return  # (shapes the operator refuses)
    batch, heads, most = src.shape
    page_size, width = cache.shape[1], block_table.shape[1] * cache.shape[1]
    dev = block_table.device
    seq = torch.arange(batch, device=dev).view(-1, 1, 1)
    head = torch.arange(heads, device=dev).view(1, -1, 1)
    src, dst = src.to(dev).long(), dst.to(dev).long()
    on = (torch.arange(most, device=dev) < counts.to(dev)[..., None]) & (src >= 0) & (src < width) & (dst >= 0) & (dst < width)

    def rows(slots):
        slots = slots.clamp(0, max(width - 1, 0))
        page = block_table[seq, slots // page_size].long() if width > 0 else slots
        return ((page * page_size + slots % page_size) * heads + head)[on]

    to = rows(dst)
    if to.unique().numel() != to.numel() or torch.isin(to, rows(src)).any():
        raise ValueError("a move's target occurs twice or is the source of a move")


def paged_kv_move(caches: Sequence[torch.Tensor], block_table: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
                  counts: torch.Tensor, *, weights: torch.Tensor | None = None,
                  slot_positions: torch.Tensor | None = None) -> None:
    """Carry out a plan's moves, in place: slot src[b, h, i] -> dst[b, h, i] for
    i < counts[b, h], in 1 to 4 caches [num_pages, page_size, Hkv, row] of any
    type (an fp16 cache's K and V, or a 4-bit cache's four tensors) and in
    weights and slot_positions. No dst may be a src or occur twice, neither by
    its slot nor by a page that two sequences name (refused with PAD_B200_CHECK=1)."""
    assert len(caches) >= 1 and all(c.is_cuda for c in caches), "pad_b200 requires CUDA tensors"
    if kernel_cuda_v4._CHECK_VALUES:
        read_error_flags(caches[0].device)
        _check_moves(caches[0], block_table, src, dst, counts)
    _OPS.kv_move(list(caches), block_table, src, dst, counts, weights, slot_positions)
    if kernel_cuda_v4._CHECK_VALUES:
        _raise_flags_of(caches[0].device)


def paged_kv_evict(caches: Sequence[torch.Tensor], weights: torch.Tensor, block_table: torch.Tensor,
                   seq_lens: torch.Tensor, budget: int, recent: int = 0, *,
                   slot_positions: torch.Tensor | None = None,
                   total_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Cut every sequence to ``budget`` slots in place (paged_kv_evict_plan, then
    paged_kv_move) and return the new seq_lens. The pages behind them are free.
    total_lens may be left out before a sequence's first eviction only (see
    paged_kv_evict_plan): from then on seq_lens is not what it has seen."""
    src, dst, counts, new_lens = paged_kv_evict_plan(weights, block_table, seq_lens, budget, recent,
                                                     slot_positions=slot_positions, total_lens=total_lens)
    paged_kv_move(caches, block_table, src, dst, counts, weights=weights, slot_positions=slot_positions)
    return new_lens
