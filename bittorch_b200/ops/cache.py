"""Operators over a decoder's key/value cache: attention of drafted tokens, eviction, beam search's selection and the
reordering of states.

A cache is a pair of tensors [B, Hkv, S, D] (float32, float16 or bfloat16, contiguous D, any other strides) with the
first ``lengths[b]`` slots of sequence b in use; ``lengths`` is an int32 or int64 tensor [B], or [1] for the whole batch,
on the device, so that a captured step can be replayed as it grows.  No function here waits for the device or keeps
anything between calls; workspaces come from the current stream's allocator.  None has a backward pass.  CUDA tensors
only, as everywhere in ``ops``.

No counterpart in the reference, whose browser runtime attends one token at a time over plain arrays
(js/src/models/TernaryTransformer.ts:366-464).
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor

from .._ext import require_ext


_bound = None


def _binding():
    global _bound
    if _bound is None:
        require_ext()
        try:
            from .. import _cache
        except ImportError as exc:
            raise RuntimeError(f"bittorch_b200: {exc}") from exc
        _bound = _cache
    return _bound


def tree_mask(parents: Tensor) -> Tensor:
    """Ancestors of every node of token trees: parents int [T] or [B, T] (the index of an earlier node, -1 for a root,
    -2 for an unused node) -> bool [T, T] or [B, T, T], ``mask[i, j]``: j is i or an ancestor of i.  Unused nodes see
    no node.  To be made once per tree shape; runs on any device."""
    if parents.dim() not in (1, 2) or parents.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"parents must be int32 or int64 [T] or [B, T], got {parents.dtype} {list(parents.shape)}")
    t = parents.shape[-1]
    node = torch.arange(t, device=parents.device)
    if bool(((parents >= node) | (parents < -2)).any()):
        raise RuntimeError("a node's parent must be an earlier node, -1 (a root) or -2 (unused)")
    unused = parents == -2
    if bool((unused.gather(-1, parents.clamp(min=0).long()) & (parents >= 0)).any()):
        raise RuntimeError("a node's parent must not be an unused node")
    mask = torch.diag_embed(~unused)
    at = parents.long()
    while bool((at >= 0).any()):
        mask |= (node == at[..., None]) & (at >= 0)[..., None]
        at = torch.where(at >= 0, parents.long().gather(-1, at.clamp(min=0)), -1)
    return mask


def tree_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, lengths: Tensor, tree: Optional[Tensor] = None,
                   scale: Optional[float] = None, mass: Optional[Tensor] = None, out: Optional[Tensor] = None) -> Tensor:
    """Attention of T new tokens per sequence, q [B, H, T, D], over a cache that already holds their keys and values in
    slots ``lengths[b] .. lengths[b] + T - 1`` -> [B, H, T, D] (laid out as [B, T, H, D]).

    Token i sees the first ``lengths[b]`` slots and the new tokens j with ``tree[i, j]`` (bool [T, T], or [B, T, T] for
    a tree per sequence; None: j <= i).  T = 1 without a tree is plain decoding.  Query head h reads key/value head
    ``h // (H // Hkv)``.  ``scale``: D ** -0.5.  A token that sees nothing gives zeros.  Slots from S on do not exist.

    Should a wait inside the kernel run out (after 2 s: a fault of the kernel or the device), what it could not write is NaN,
    and ``_C.device_status()`` says so.

    ``mass`` float32 [B, Hkv, S]: every slot's attention weight, summed over the heads of its group and the T tokens, is
    added to it in place (what ``evict_cache`` goes by)."""
    return _binding().tree_attention(q, k_cache, v_cache, lengths, tree, scale, mass, out)


def evict_select(mass: Tensor, lengths: Tensor, budget: int, sinks: int, recent: int) -> Tuple[Tensor, Tensor]:
    """Which slots of a cache stay: per sequence and key/value head the first ``sinks`` slots, the last ``recent``, and
    of the others those with the largest accumulated weight ``mass`` [B, Hkv, S] (equal weights: the lowest slot),
    ``budget`` in all.  -> (keep int64 [B, Hkv, budget], slots in order, -1 from ``counts[b]`` on; counts int64 [B], the
    new lengths).  A sequence of at most ``budget`` slots keeps them all."""
    return _binding().evict_select(mass, lengths, budget, sinks, recent)


def compact_cache(k_cache: Tensor, v_cache: Tensor, keep: Tensor, counts: Tensor, first: Optional[Tensor] = None,
                  mass: Optional[Tensor] = None, out: Optional[Sequence[Tensor]] = None) -> None:
    """Moves cache slots together: slot ``first[b] + j`` takes slot ``keep[b, h, j]`` for j < ``counts[b]`` (``first``
    int64 [B], None: 0; ``keep`` int64 [B, Hkv or 1, n]).  In place, where ``keep`` has to ascend with ``keep[b, h, j]
    >= first[b] + j``, or into ``out`` = (keys, values[, mass]) of any number of slots.  ``mass`` is moved like the rows
    and set to zero behind them.  Entries of ``keep`` outside the cache are skipped."""
    _binding().compact_cache(k_cache, v_cache, keep, counts, first, mass, out)


def evict_cache(k_cache: Tensor, v_cache: Tensor, mass: Tensor, lengths: Tensor, budget: int, sinks: int = 4,
                recent: int = 0, out: Optional[Sequence[Tensor]] = None) -> Tuple[Tensor, Tensor]:
    """Cuts a cache down to ``budget`` slots per sequence and head: ``evict_select``, then ``compact_cache`` of keys, values
    and mass, in place or into ``out`` = (keys, values, mass) with at least ``budget`` slots.  -> (keep, counts)."""
    return _binding().evict_cache(k_cache, v_cache, mass, lengths, budget, sinks, recent, out)


def beam_select(logits: Tensor, scores: Tensor, select: Optional[int] = None, finished: Optional[Tensor] = None,
                end_token: Optional[int] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """The ``select`` best continuations (default: as many as beams) of every sequence by ``scores[b, w] +
    log_softmax(logits[b, w])[v]``, best first; equal scores go to the lowest ``w * V + v``.  Sums are ranked in float64; a
    row's log-sum of exponentials in them is off by 3.3e-6 at most (float32 exponentials; 2e-7 as a rule), so that candidates
    of different beams that are closer than this may change places.
    logits [B, beams, V], scores float32 [B, beams].  A beam with ``finished[b, w]`` goes on by ``end_token`` alone, its
    score unchanged.  NaN logits, and beams without a finite score or a finite largest logit, count as -infinity.
    -> (scores float32, tokens int64, parents int64), each [B, select]."""
    return _binding().beam_select(logits, scores, select, finished, end_token)


def reorder_cache(caches: Sequence[Tensor], parents: Tensor, lengths: Tensor, start: int = 0) -> None:
    """Gives every beam its parent's states, in place, in one launch: for every tensor [B * beams, Hkv, S, D] of
    ``caches`` (the keys and values of all layers), slots ``start .. lengths[b] - 1`` of row ``b * beams + w`` become
    those that row ``b * beams + parents[b, w]`` had.  ``start``: slots that all beams share (a prompt).  ``lengths``
    is per sequence [B] or [1].  A parent outside the beams leaves its row as it is."""
    _binding().reorder_cache(caches, parents, lengths, start)
