"""Layers on the invariant channels of nodes: ``Embedding`` of their kinds, ``SegmentAttention`` among the nodes of a
structure and the ``GatedFeedForward`` block."""
from typing import Optional

import torch
from torch import Tensor, nn

from .functional.attention import AttentionPlan, segment_attention
from .functional.embedding import embedding
from .functional.feed_forward import _ACTIVATIONS, gated_feed_forward
from .init import initialize_linear


class Embedding(nn.Module):
    """``kind`` int64 of any shape -> ``(*kind.shape, channels)``, rows of a learnable ``(kinds, channels)`` table times
    ``scale``; a kind outside the table gives zeros."""

    def __init__(self, kinds: int, channels: int, scale: float = 1.0):
        super().__init__()
        if kinds < 1 or channels < 1:
            raise ValueError(f"kinds and channels must be positive, got {kinds} and {channels}")
        self.kinds, self.channels, self.scale = kinds, channels, scale
        self.weight = nn.Parameter(torch.empty(kinds, channels))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        nn.init.normal_(self.weight)

    def forward(self, kind: Tensor) -> Tensor:
        return embedding(kind, self.weight, self.scale)

    def extra_repr(self) -> str:
        return f"kinds={self.kinds}, channels={self.channels}, scale={self.scale}"


class SegmentAttention(nn.Module):
    """Attention of every node over the nodes of its own structure, ``(N, channels) -> (N, channels)``, or of queries over
    other nodes (``x_k``, with a plan that has ``ptr_k``): a readout.  ``heads`` query heads of ``channels // heads``
    channels share ``kv_heads`` heads of keys and values.  ``cap`` bounds the scores, ``cap * tanh(score / cap)``.

    ``distances``: a learnable multiple of the distance, one for each query head (``2 ** (-8 (h + 1) / heads)`` at first),
    is taken off the score; ``pos`` (and ``pos_k``) are fp32 and get gradients."""

    def __init__(self, channels: int, heads: int, kv_heads: Optional[int] = None, cap: Optional[float] = None,
                 distances: bool = True):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads < 1 or channels % heads or not 1 <= channels // heads <= 128:
            raise ValueError(f"channels must be heads times 1 .. 128, got {channels} and {heads}")
        if kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"heads must be a multiple of kv_heads, got {heads} and {kv_heads}")
        self.channels, self.heads, self.kv_heads, self.cap, self.distances = channels, heads, kv_heads, cap, distances
        self.head_channels = channels // heads
        self.weight_in = nn.Parameter(torch.empty(channels, (heads + 2 * kv_heads) * self.head_channels))
        self.weight_out = nn.Parameter(torch.empty(channels, channels))
        if distances:
            self.slope = nn.Parameter(torch.empty(heads))
        else:
            self.register_parameter("slope", None)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        initialize_linear(self.weight_in)
        initialize_linear(self.weight_out)
        if self.slope is not None:
            with torch.no_grad():
                self.slope.copy_(torch.exp2(torch.arange(1, self.heads + 1) * (-8.0 / self.heads)))

    def forward(self, x: Tensor, plan: AttentionPlan, pos: Optional[Tensor] = None, x_k: Optional[Tensor] = None,
                pos_k: Optional[Tensor] = None) -> Tensor:
        if (pos is not None) != self.distances:
            raise ValueError("pos is given exactly where distances are used")
        h, hk, d = self.heads, self.kv_heads, self.head_channels
        if x_k is None:
            q, k, v = (x @ self.weight_in).view(-1, h + 2 * hk, d).split((h, hk, hk), 1)
        else:
            q = (x @ self.weight_in[:, :h * d]).view(-1, h, d)
            k, v = (x_k @ self.weight_in[:, h * d:]).view(-1, 2 * hk, d).split((hk, hk), 1)
        slope = None if self.slope is None else self.slope.float()
        out = segment_attention(q, k, v, plan, pos, slope, pos_k, self.cap)
        return out.view(-1, self.channels) @ self.weight_out

    def extra_repr(self) -> str:
        return (f"channels={self.channels}, heads={self.heads}, kv_heads={self.kv_heads}, cap={self.cap}, "
                f"distances={self.distances}")


class GatedFeedForward(nn.Module):
    """``(act(x Wg) * (x Wu)) Wd`` over the last axis, ``channels -> hidden -> channels_out`` (``channels`` unless given);
    ``activation`` ``"silu"``, ``"gelu"`` or ``"sigmoid"``."""

    def __init__(self, channels: int, hidden: int, channels_out: Optional[int] = None, activation: str = "silu"):
        super().__init__()
        channels_out = channels if channels_out is None else channels_out
        if min(channels, hidden, channels_out) < 1:
            raise ValueError(f"channels must be positive, got {channels}, {hidden} and {channels_out}")
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
        self.channels, self.hidden, self.channels_out, self.activation = channels, hidden, channels_out, activation
        self.weight_gate = nn.Parameter(torch.empty(channels, hidden))
        self.weight_up = nn.Parameter(torch.empty(channels, hidden))
        self.weight_down = nn.Parameter(torch.empty(hidden, channels_out))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        for weight in (self.weight_gate, self.weight_up, self.weight_down):
            initialize_linear(weight)

    def forward(self, x: Tensor) -> Tensor:
        return gated_feed_forward(x, self.weight_gate, self.weight_up, self.weight_down, self.activation)

    def extra_repr(self) -> str:
        return (f"channels={self.channels}, hidden={self.hidden}, channels_out={self.channels_out}, "
                f"activation='{self.activation}'")
