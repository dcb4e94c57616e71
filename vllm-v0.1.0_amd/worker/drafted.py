"""Host side of checking drafted tokens over the paged cache.

A step that checks drafts puts the drafted tokens' keys and values behind each sequence's context
(cache_ops.reshape_and_cache, slots context_len - T ... context_len - 1 in the order of their rows), runs
attention_ops.tree_cached_kv_attention with the mask of the trees, and keeps the accepted path: its
tokens move to consecutive slots, and the context ends behind them.  No counterpart in the reference.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np
import torch


def tree_mask(parents: Sequence[Sequence[int]], device: torch.device | str = "cuda") -> torch.Tensor:
    """The mask attention_ops.tree_cached_kv_attention takes, from the trees' parents: parents[s][i] is the
    drafted token of sequence s that its i-th one follows (an earlier one), or -1 where it follows the
    context.  A token sees itself and its ancestors.  bool [sum of lengths, longest length]."""
    width = max((len(p) for p in parents), default=0)
    mask = np.zeros((sum(len(p) for p in parents), max(width, 1)), dtype=bool)
    row = 0
    for p in parents:
        for i, parent in enumerate(p):
            if not -1 <= parent < i:
                raise ValueError(f"token {i}'s parent ({parent}) must be an earlier token, or -1")
            if parent >= 0:
                mask[row + i] = mask[row + parent]
            mask[row + i, i] = True
        row += len(p)
    return torch.from_numpy(mask).to(device)


def keep_path(key_caches: List[torch.Tensor], value_caches: List[torch.Tensor], block_tables: torch.Tensor,
              first_positions: Sequence[int], paths: Sequence[Sequence[int]], cache_ops=None,
              weight_caches: Optional[List[torch.Tensor]] = None) -> None:
    """Moves every sequence's accepted drafted tokens, paths[s] (rising indices into its draft), to the
    consecutive positions from first_positions[s] on (the context length without the draft), in all layers.
    Tokens already in place are not touched; the moves of one layer are one gather and one scatter.

    weight_caches, one per layer, where weights are accumulated for cache_ops.evict_cached_kv: the accepted
    positions' entries start from 0.  Attention of a tree gives its tokens no weights, and an entry holds whatever
    its block did before it was handed out, which an eviction would take for a weight."""
    if cache_ops is None:
        from .. import cache_ops  # HIP module; no fallback
    if len(paths) > block_tables.shape[0] or len(paths) > len(first_positions):
        raise ValueError(f"{len(paths)} paths for a block table of {block_tables.shape[0]} sequences, {len(first_positions)} positions")
    if weight_caches is not None:
        if len(weight_caches) != len(value_caches):
            raise ValueError(f"{len(weight_caches)} weight caches for {len(value_caches)} layers")
        for wc, vc in zip(weight_caches, value_caches):
            if tuple(wc.shape) != (vc.shape[0], vc.shape[1], vc.shape[3]):
                raise ValueError(f"a weight cache must be [num_blocks, num_kv_heads, block_size] like its value cache, is {list(wc.shape)}")
    moved, in_place = [], []  # (sequence, from, to)
    for s, path in enumerate(paths):
        for i, t in enumerate(path):
            if i and t <= path[i - 1] or t < 0:
                raise ValueError(f"the path of sequence {s} must rise: {list(path)}")
            (in_place if t == i else moved).append((s, first_positions[s] + t, first_positions[s] + i))
    touched = moved if weight_caches is None else moved + in_place
    if not touched:
        return
    block = value_caches[0].shape[3]
    low, high = min(to for _, _, to in touched), max(at for _, at, _ in touched)
    if low < 0 or high >= block_tables.shape[1] * block:
        raise ValueError(f"a path runs from position {low} to {high}, the block tables hold {block_tables.shape[1] * block}")
    device = block_tables.device
    sequence, *places = torch.tensor(touched, dtype=torch.int64, device=device).t()
    source, target = ((block_tables[sequence, at // block].long(), at % block) for at in places)
    if weight_caches is not None:
        for wc in weight_caches:
            wc[target[0], :, target[1]] = 0.0
    if not moved:
        return
    n = len(moved)
    slots = [(b[:n] * block + o[:n]).int() for b, o in (source, target)]
    heads, dim = value_caches[0].shape[1:3]
    key = torch.empty(n, heads, dim, dtype=value_caches[0].dtype, device=device)
    value = torch.empty_like(key)
    for kc, vc in zip(key_caches, value_caches):
        cache_ops.gather_cached_kv(key, value, kc, vc, slots[0])
        cache_ops.reshape_and_cache(key, value, kc, vc, slots[1])
