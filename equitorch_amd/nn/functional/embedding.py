"""Embedding of node kinds (species, local environments) into invariant channels.

The lookup and its gradient are one call of the library each: ``cgtp_embed_forward`` and ``cgtp_embed_backward``, which
sorts the rows by kind and sums them in an order that does not depend on timing."""
import torch
from torch import Tensor
from torch.autograd import Function

from ... import _lib, _shim
from ..._lib import CgtpError


def _lookup(kind: Tensor, table: Tensor, scale: float) -> Tensor:
    kinds, c = table.shape
    out = torch.empty((*kind.shape, c), dtype=table.dtype, device=table.device)
    _lib.check(_lib.lib.cgtp_embed_forward(kind.data_ptr(), table.data_ptr(), out.data_ptr(), kind.numel(), kinds, c, scale,
                                           _lib.dtype_code(table.dtype), _lib.stream_ptr(table.device)),
               "cgtp_embed_forward")
    return out


class _Embedding(Function):
    @staticmethod
    def forward(ctx, kind: Tensor, table: Tensor, scale: float):
        ctx.save_for_backward(kind)
        ctx.scale, ctx.kinds = scale, table.shape[0]
        return _lookup(kind, table, scale)

    @staticmethod
    def backward(ctx, g):
        (kind,) = ctx.saved_tensors
        return None, _EmbeddingGrad.apply(kind, g, ctx.kinds, ctx.scale), None


class _EmbeddingGrad(Function):
    """The gradient is linear in ``g``; its own gradient is the lookup again."""

    @staticmethod
    def forward(ctx, kind: Tensor, g: Tensor, kinds: int, scale: float):
        ctx.save_for_backward(kind)
        ctx.scale = scale
        g = g.contiguous()
        c, n = g.shape[-1], kind.numel()
        out = torch.empty((kinds, c), dtype=g.dtype, device=g.device)
        code = _lib.dtype_code(g.dtype)
        ws = torch.empty(_lib.lib.cgtp_embed_workspace_bytes(n, kinds, c, code), dtype=torch.uint8, device=g.device)
        _lib.check(_lib.lib.cgtp_embed_backward(kind.data_ptr(), g.data_ptr(), out.data_ptr(), ws.data_ptr(), n, kinds, c,
                                                scale, code, _lib.stream_ptr(g.device)), "cgtp_embed_backward")
        return out

    @staticmethod
    def backward(ctx, gg):
        (kind,) = ctx.saved_tensors
        return None, _Embedding.apply(kind, gg.contiguous(), ctx.scale), None, None


def embedding(kind: Tensor, table: Tensor, scale: float = 1.0) -> Tensor:
    """``out[..., c] = scale * table[kind[...], c]``: ``kind`` int64 of any shape, ``table`` ``(kinds, C)`` in fp32, fp64,
    bf16 or fp16.  A kind outside the table gives a row of zeros and no gradient (no check on the host, which would wait
    for the GPU).  The gradient of ``table`` is summed in 32 bits (64 for fp64) and rounded once; differentiable to any
    order."""
    _lib.require_gpu(kind, table)
    if kind.dtype != torch.int64:
        raise CgtpError(f"kind must be int64, got {kind.dtype}")
    if table.ndim != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise CgtpError(f"table must be (kinds, C) with at least one of each, got {tuple(table.shape)}")
    if kind.device != table.device:
        raise CgtpError(f"kind is on {kind.device}, table on {table.device}")
    _lib.dtype_code(table.dtype)
    kind, table = kind.contiguous(), table.contiguous()
    mod = _shim.module()
    if mod is not None:
        return mod.embed(kind, table, float(scale))
    if (torch.is_grad_enabled() and table.requires_grad) or _lib.forward_mode():
        return _Embedding.apply(kind, table, float(scale))
    return _lookup(kind, table, float(scale))
