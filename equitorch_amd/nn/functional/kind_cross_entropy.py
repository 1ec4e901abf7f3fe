"""Softmax cross entropy over the kinds of a table, on invariant channels.

    z = scale x table^T  (cap: cap tanh(scale x table^T / cap)),  loss = log sum_k exp z_k - z_kind

``cgtp_kind_loss_forward`` and ``cgtp_kind_loss_backward`` take the table in pieces and never keep the logits; gradients of
higher order are taken through the tensor expression, which does."""
import ctypes as C
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import Function

from ... import _lib, _shim
from ..._lib import CgtpError, KindLossArgs
from ._higher_order import higher_order

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _args(x: Tensor, table: Tensor, kind: Tensor, scale: float, cap: float) -> KindLossArgs:
    a = KindLossArgs()
    a.x, a.table, a.kind = x.data_ptr(), table.data_ptr(), kind.data_ptr()
    a.n_rows, a.n_kinds, a.channels, a.dtype = x.shape[0], table.shape[0], x.shape[1], _lib.dtype_code(x.dtype)
    a.scale, a.cap = scale, cap
    return a


def _launch(a: KindLossArgs, backward: int, x: Tensor) -> None:
    ws = torch.empty(_lib.lib.cgtp_kind_loss_workspace_bytes(C.byref(a), backward), dtype=torch.uint8, device=x.device)
    a.workspace = ws.data_ptr()
    name = "cgtp_kind_loss_backward" if backward else "cgtp_kind_loss_forward"
    with torch.cuda.device(x.device):
        _lib.check(getattr(_lib.lib, name)(C.byref(a), _lib.stream_ptr(x.device)), name)


def _forward(x: Tensor, table: Tensor, kind: Tensor, scale: float, cap: float, keep: bool):
    """``(loss, lse)``, lse None unless ``keep``."""
    loss = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    lse = torch.empty_like(loss) if keep else None
    a = _args(x, table, kind, scale, cap)
    a.loss, a.lse = loss.data_ptr(), _lib.ptr(lse)
    _launch(a, 0, x)
    return loss, lse


def _higher(g: Tensor, inputs, need, kind: Tensor, scale: float, cap: float):
    def expression(x, table):
        asked = ((kind >= 0) & (kind < table.shape[0])).nonzero()[:, 0]
        z = x[asked].float() @ table.float().T * scale
        if cap:
            z = cap * torch.tanh(z / cap)
        at = z.gather(1, kind[asked, None])[:, 0]
        loss = torch.zeros(x.shape[0], dtype=torch.float32, device=x.device)
        return loss.index_put((asked,), torch.logsumexp(z, 1) - at)
    return higher_order(expression, inputs, need, g)


_fallbacks = []


def _fallback(mod):
    """The extension's number for the tensor expression, which a backward under gradient mode evaluates."""
    if not _fallbacks:
        _fallbacks.append(mod.Fallback(_higher))
    return _fallbacks[0]


class _KindCrossEntropy(Function):
    @staticmethod
    def forward(ctx, x: Tensor, table: Tensor, kind: Tensor, scale: float, cap: float):
        loss, lse = _forward(x, table, kind, scale, cap, True)
        ctx.save_for_backward(x, table, kind, lse)
        ctx.scale, ctx.cap = scale, cap
        return loss

    @staticmethod
    def backward(ctx, g):
        x, table, kind, lse = ctx.saved_tensors
        need = ctx.needs_input_grad[:2]
        if torch.is_grad_enabled():
            return (*_higher(g, (x, table), need, kind, ctx.scale, ctx.cap), None, None, None)
        g = g.contiguous()
        grads = [torch.empty_like(t) if n else None for t, n in zip((x, table), need)]
        a = _args(x, table, kind, ctx.scale, ctx.cap)
        a.lse, a.grad_loss, a.grad_x, a.grad_table = lse.data_ptr(), g.data_ptr(), _lib.ptr(grads[0]), _lib.ptr(grads[1])
        _launch(a, 1, x)
        return (*grads, None, None, None)


def kind_cross_entropy(x: Tensor, table: Tensor, kind: Tensor, scale: float = 1.0, cap: Optional[float] = None) -> Tensor:
    """``loss[...] = log sum_k exp z[..., k] - z[..., kind[...]]`` in fp32 with ``z = scale * x @ table.T``, or ``cap * tanh(scale * x @
    table.T / cap)``: ``x`` ``(..., C)``, ``table`` ``(kinds, C)`` (an :func:`embedding`'s, say), both fp32, bf16 or fp16 (under
    autocast also mixed: autocast's type), ``kind`` int64 ``(...)``.

    Where ``kind`` is outside the table the loss is 0 and nothing has a gradient, whatever ``x`` holds there: nodes that are not
    asked for have kind -1 and cost nothing.  No logits are kept.  Sums are held in 32 bits and have a fixed order; the
    softmax is rounded to the operands' type where it enters the gradients' products, and for the table's so are the rows of ``x`` times
    the incoming gradient over its largest magnitude (in fp16 rows whose gradient is below some 1e-5 of that keep few bits)."""
    tensors = x, table = _lib.of_one_type(x, table)
    _lib.require_gpu(x, table, kind)
    if x.dtype not in _DTYPES or table.dtype != x.dtype:
        raise CgtpError(f"x and table must be fp32, bf16 or fp16, of one type, got {x.dtype} and {table.dtype}")
    if kind.dtype != torch.int64:
        raise CgtpError(f"kind must be int64, got {kind.dtype}")
    if table.device != x.device or kind.device != x.device:
        raise CgtpError(f"operands are on different devices: {x.device}, {table.device}, {kind.device}")
    c = x.shape[-1] if x.ndim else 0
    if not 1 <= c < 1 << 15 or table.ndim != 2 or table.shape[0] < 1 or table.shape[1] != c or kind.shape != x.shape[:-1]:
        raise CgtpError(f"shapes must be x (..., C) with 1 <= C < 2^15, table (kinds, C), kind (...), got {tuple(x.shape)}, "
                        f"{tuple(table.shape)}, {tuple(kind.shape)}")
    scale, bounded = float(scale), cap is not None
    cap = float(cap) if bounded else 0.0
    # the kernels take scale * log2 e, or scale / cap and cap * log2 e, as fp32, where a quotient below the normal numbers loses its bits, or is zero
    least = 2.0 ** -126 if scale else 0.0
    if not least <= abs(scale) <= 1e38 or (bounded and not (1e-37 <= cap <= 1e38 and least <= abs(scale) / cap <= 1e38)):
        raise CgtpError(f"scale, cap (above zero, or None) and their quotient must be in fp32's range, got {scale} and {cap}")
    if (x.numel() and kind.numel() > 1 << 29) or table.shape[0] > 1 << 30:
        raise CgtpError(f"at most 2^29 rows and 2^30 kinds, got {kind.numel()} and {table.shape[0]}")
    flat, table, kinds = x.reshape(-1, c).contiguous(), table.contiguous(), kind.reshape(-1).contiguous()
    keep = (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)) or _lib.forward_mode()
    mod = _shim.module()
    if mod is not None:
        loss = mod.kind_loss(flat, table, kinds, scale, cap, keep, _fallback(mod))
    elif keep:
        loss = _KindCrossEntropy.apply(flat, table, kinds, scale, cap)
    else:
        loss = _forward(flat, table, kinds, scale, cap, False)[0]
    return loss if x.ndim == 2 else loss.reshape(kind.shape)
