"""Host side of checking drafted tokens over the paged cache.

A step that checks drafts puts the drafted tokens' keys and values behind each sequence's context
(cache_ops.reshape_and_cache, slots context_len - T ... context_len - 1 in the order of their rows), runs
attention_ops.tree_cached_kv_attention with the mask of the trees, and keeps the accepted path: its
tokens move to consecutive slots, and the context ends behind them.  No counterpart in the reference.
"""
from __future__ import annotations

from typing import List, Sequence

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
              first_positions: Sequence[int], paths: Sequence[Sequence[int]], cache_ops=None) -> None:
    """Moves every sequence's accepted drafted tokens, paths[s] (rising indices into its draft), to the
    consecutive positions from first_positions[s] on (the context length without the draft), in all layers.
    Tokens already in place are not touched; the moves of one layer are one gather and one scatter."""
    if cache_ops is None:
        from .. import cache_ops  # HIP module; no fallback
    if len(paths) > block_tables.shape[0] or len(paths) > len(first_positions):
        raise ValueError(f"{len(paths)} paths for a block table of {block_tables.shape[0]} sequences, {len(first_positions)} positions")
    sequence, source, target = [], [], []
    for s, path in enumerate(paths):
        for i, t in enumerate(path):
            if i and t <= path[i - 1] or t < 0:
                raise ValueError(f"the path of sequence {s} must rise: {list(path)}")
            if t != i:
                sequence.append(s)
                source.append(first_positions[s] + t)
                target.append(first_positions[s] + i)
    if not sequence:
        return
    block = value_caches[0].shape[3]
    if min(target) < 0 or max(source) >= block_tables.shape[1] * block:
        raise ValueError(f"a path runs from position {min(target)} to {max(source)}, the block tables hold {block_tables.shape[1] * block}")
    device = block_tables.device
    seq, src, dst = (torch.tensor(x, dtype=torch.int64, device=device) for x in (sequence, source, target))
    slots = [(block_tables[seq, at // block].long() * block + at % block).int() for at in (src, dst)]
    heads, dim = value_caches[0].shape[1:3]
    key = torch.empty(len(sequence), heads, dim, dtype=value_caches[0].dtype, device=device)
    value = torch.empty_like(key)
    for kc, vc in zip(key_caches, value_caches):
        cache_ops.gather_cached_kv(key, value, kc, vc, slots[0])
        cache_ops.reshape_and_cache(key, value, kc, vc, slots[1])
