"""Gated feed-forward block on invariant channels.

    g = x Wg,  u = x Wu,  out = (act(g) * u) Wd

``cgtp_gff_forward`` and ``cgtp_gff_backward`` do the whole block, one call each way; gradients of higher order are taken
through the tensor expression."""
import ctypes as C

import torch
from torch import Tensor
from torch.autograd import Function

from ... import _lib, _shim
from ..._lib import CgtpError, GffArgs
from ._higher_order import higher_order

_ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2}
_EXPRESSIONS = (torch.nn.functional.silu, torch.nn.functional.gelu, torch.sigmoid)
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _args(x, w_gate, w_up, w_down, mid, code, act) -> GffArgs:
    a = GffArgs()
    a.x, a.w_gate, a.w_up, a.w_down, a.mid = x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), mid.data_ptr()
    a.n_rows, a.c_in, a.hidden, a.c_out = x.shape[0], x.shape[1], w_gate.shape[1], w_down.shape[1]
    a.activation, a.dtype = act, code
    return a


def _forward(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, act: int, keep: bool):
    """``(out, gate, up, mid)``; gate and up are None unless ``keep``."""
    n, h = x.shape[0], (w_gate.shape[1] + 7) // 8 * 8
    out = torch.empty((n, w_down.shape[1]), dtype=x.dtype, device=x.device)
    if keep:
        gate, up, mid = torch.empty((3, n, h), dtype=x.dtype, device=x.device)
    else:
        gate, up, mid = None, None, torch.empty((n, h), dtype=x.dtype, device=x.device)
    a = _args(x, w_gate, w_up, w_down, mid, _lib.dtype_code(x.dtype), act)
    a.out, a.gate, a.up = out.data_ptr(), _lib.ptr(gate), _lib.ptr(up)
    nbytes = _lib.lib.cgtp_gff_workspace_bytes(C.byref(a), 0)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    a.workspace = _lib.ptr(ws)
    _lib.check(_lib.lib.cgtp_gff_forward(C.byref(a), _lib.stream_ptr(x.device)), "cgtp_gff_forward")
    return out, gate, up, mid


def _expression(act: int):
    fn = _EXPRESSIONS[act]

    def expression(x, wg, wu, wd):
        dtype = x.dtype
        x, wg, wu, wd = (t.float() for t in (x, wg, wu, wd))
        return ((fn(x @ wg) * (x @ wu)) @ wd).to(dtype)
    return expression


_fallbacks = {}


def _fallback(mod, act: int):
    """The extension's number for the tensor expression of an activation, which a backward under gradient mode evaluates."""
    if act not in _fallbacks:
        _fallbacks[act] = mod.Fallback(lambda g, inputs, need: higher_order(_expression(act), inputs, need, g))
    return _fallbacks[act]


class _GatedFeedForward(Function):
    @staticmethod
    def forward(ctx, x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, act: int):
        out, gate, up, mid = _forward(x, w_gate, w_up, w_down, act, True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, gate, up, mid)
        ctx.act = act
        return out

    @staticmethod
    def backward(ctx, g):
        x, w_gate, w_up, w_down, gate, up, mid = ctx.saved_tensors
        need = ctx.needs_input_grad[:4]
        if torch.is_grad_enabled():
            return (*higher_order(_expression(ctx.act), (x, w_gate, w_up, w_down), need, g), None)
        g = g.contiguous()
        grads = [torch.empty_like(t) if n else None for t, n in zip((x, w_gate, w_up, w_down), need)]
        g_gate, g_up = torch.empty((2, *mid.shape), dtype=x.dtype, device=x.device)
        a = _args(x, w_gate, w_up, w_down, mid, _lib.dtype_code(x.dtype), ctx.act)
        a.gate, a.up, a.grad_out = gate.data_ptr(), up.data_ptr(), g.data_ptr()
        a.grad_gate, a.grad_up = g_gate.data_ptr(), g_up.data_ptr()
        a.grad_x, a.grad_w_gate, a.grad_w_up, a.grad_w_down = (_lib.ptr(t) for t in grads)
        ws = torch.empty(_lib.lib.cgtp_gff_workspace_bytes(C.byref(a), 1), dtype=torch.uint8, device=x.device)
        a.workspace = ws.data_ptr()
        _lib.check(_lib.lib.cgtp_gff_backward(C.byref(a), _lib.stream_ptr(x.device)), "cgtp_gff_backward")
        return (*grads, None)


def gated_feed_forward(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, activation: str = "silu") -> Tensor:
    """``(act(x w_gate) * (x w_up)) w_down`` over the last axis of ``x``: ``x`` ``(..., C_in)``, ``w_gate`` and ``w_up``
    ``(C_in, H)``, ``w_down`` ``(H, C_out)``, all fp32, bf16 or fp16 (under autocast also mixed: autocast's type); ``activation`` ``"silu"``, ``"gelu"`` (with the error
    function) or ``"sigmoid"``.

    Products and activation are computed in 32 bits.  What is kept between the products — ``act(x w_gate) * (x w_up)``,
    and for a backward pass the two projections and their gradients — is rounded to the operands' type, so in fp16 it has
    fp16's range.  Gradients of the weights are summed over the rows in a fixed order."""
    tensors = x, w_gate, w_up, w_down = _lib.of_one_type(x, w_gate, w_up, w_down)
    _lib.require_gpu(*tensors)
    if activation not in _ACTIVATIONS:
        raise CgtpError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if x.dtype not in _DTYPES or any(t.dtype != x.dtype for t in tensors):
        raise CgtpError(f"operands must be fp32, bf16 or fp16, all of one type, got {[str(t.dtype) for t in tensors]}")
    if any(t.device != x.device for t in tensors):
        raise CgtpError(f"operands are on different devices: {[str(t.device) for t in tensors]}")
    c = x.shape[-1] if x.ndim else 0
    if x.ndim < 1 or w_gate.ndim != 2 or w_gate.shape[0] != c or w_up.shape != w_gate.shape or w_down.ndim != 2 \
            or w_down.shape[0] != w_gate.shape[1] or 0 in (*w_gate.shape, *w_down.shape):
        raise CgtpError(f"shapes must be x (..., C_in), w_gate and w_up (C_in, H), w_down (H, C_out), got "
                        f"{[tuple(t.shape) for t in tensors]}")
    flat = x.reshape(-1, c).contiguous()
    weights = [t.contiguous() for t in (w_gate, w_up, w_down)]
    act = _ACTIVATIONS[activation]
    keep = (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)) or _lib.forward_mode()
    mod = _shim.module()
    if mod is not None:
        out = mod.gff(flat, *weights, act, keep, _fallback(mod, act))
    elif keep:
        out = _GatedFeedForward.apply(flat, *weights, act)
    else:
        out = _forward(flat, *weights, act, False)[0]
    return out if x.ndim == 2 else out.reshape(*x.shape[:-1], w_down.shape[1])
