"""Rotary positions in both pair layouts, over part of a head, stretched for long contexts, with head norms.

The reference has one rotation (PagedAttentionWithRoPE, vllm/model_executor/layers/attention.py:159-215:
half layout, table in the default dtype, its rounding after every operation).  This module drives the
two operators next to it, pos_encoding_ops.rotary_embedding and qk_norm_rotary_embedding, which compute
in fp32 from a float32 table and round once.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn


def rotary_cos_sin_cache(rotary_dim: int, max_position: int, base: float = 10000.0, scaling: str = "none",
                         factor: float = 1.0, original_max_position: Optional[int] = None, fast_turns: float = 32.0,
                         slow_turns: float = 1.0, device: torch.device | str = "cpu") -> torch.Tensor:
    """The [max_position, rotary_dim] float32 table (cos half, sin half) that the rotary operators take.

    Pair i turns by position * base^(-2 i / rotary_dim).  Angles are made in float64: at position 10^5 a
    float32 product is already off by 10^-2 of a radian.  `scaling` stretches a model trained to
    `original_max_position` (default max_position / factor) by `factor`:

      "none"    nothing
      "linear"  every position divided by factor
      "ntk"     base * factor^(d / (d - 2)): the slowest pair is stretched by factor, the fastest not
      "yarn"    pairs of over fast_turns turns within the original length as they are, of under
                slow_turns divided by factor, a ramp over the pair index between; cos and sin times
                0.1 ln(factor) + 1, which keeps the entropy of the attention weights
    """
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim ({rotary_dim}) must be even.")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"Rotary scaling {scaling!r} is not supported.")
    if not factor >= 1.0:
        raise ValueError(f"Rotary scaling factor ({factor}) must be at least 1.")
    pair = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    amplitude = 1.0
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freq = torch.pow(torch.tensor(base, dtype=torch.float64, device=device), -pair / max(rotary_dim, 1))
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        length = original_max_position if original_max_position is not None else max_position / factor
        # the pair that turns `turns` times within the original length
        low, high = (rotary_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))
                     for turns in (fast_turns, slow_turns))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rotary_dim - 1)
        ramp = ((pair / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * (1 - ramp) + freq / factor * ramp
        amplitude = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(max_position, dtype=torch.float64, device=device)[:, None] * freq[None]
    return torch.cat((angle.cos() * amplitude, angle.sin() * amplitude), dim=1).float()


class RotaryEmbedding(nn.Module):
    """Rotates query and key in place: [num_tokens, num_heads * head_size] and [num_tokens, num_kv_heads *
    head_size] rows, column slices of a fused projection among them.  With qk_norm every head is RMS-normed
    first, in the same pass (query_weight, key_weight: [head_size])."""

    def __init__(self, head_size: int, rotary_dim: int, max_position: int = 8192, base: float = 10000.0,
                 interleaved: bool = False, scaling: str = "none", factor: float = 1.0,
                 original_max_position: Optional[int] = None, qk_norm: bool = False, eps: float = 1e-6,
                 pos_encoding_ops=None) -> None:
        super().__init__()
        if pos_encoding_ops is None:
            from .. import pos_encoding_ops  # HIP module; no fallback
        self._pos_encoding_ops = pos_encoding_ops
        self.head_size = head_size
        self.interleaved = interleaved
        self.variance_epsilon = eps
        table = rotary_cos_sin_cache(rotary_dim, max_position, base, scaling, factor, original_max_position)
        self.register_buffer("cos_sin_cache", table, persistent=False)
        self.query_weight = nn.Parameter(torch.ones(head_size)) if qk_norm else None
        self.key_weight = nn.Parameter(torch.ones(head_size)) if qk_norm else None

    def _apply(self, fn, recurse=True):
        # .half(), .to(dtype) and .to_empty() are meant for the weights, which a checkpoint fills: the table keeps its
        # numbers, and follows the device to where they can be
        table = self.cos_sin_cache
        super()._apply(fn, recurse)
        device = self.cos_sin_cache.device
        self.cos_sin_cache = table if device.type == "meta" else table.to(device)
        return self

    def forward(self, positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor) -> None:
        if self.query_weight is None:
            self._pos_encoding_ops.rotary_embedding(positions, query, key, self.head_size, self.cos_sin_cache, self.interleaved)
        else:
            self._pos_encoding_ops.qk_norm_rotary_embedding(positions, query, key, self.head_size, self.query_weight.data,
                                                            self.key_weight.data, self.variance_epsilon, self.cos_sin_cache,
                                                            self.interleaved)
