"""Root-mean-square norm after a residual's addition, on invariant channels.

    total = x + residual,  out = total * weight / sqrt(mean_c total^2 + eps)

``cgtp_add_rms_forward`` and ``cgtp_add_rms_backward`` do both and their gradients, one call each way; gradients of higher
order are taken through the tensor expression."""
import ctypes as C
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import Function

from ... import _lib, _shim
from ..._lib import AddRmsArgs, CgtpError
from ._higher_order import higher_order

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _args(x: Tensor, weight: Optional[Tensor], total_type: torch.dtype, eps: float) -> AddRmsArgs:
    a = AddRmsArgs()
    a.weight, a.n_rows, a.channels, a.eps = _lib.ptr(weight), x.shape[0], x.shape[1], eps
    a.dtype, a.residual_dtype = _lib.dtype_code(x.dtype), _lib.dtype_code(total_type)
    a.weight_dtype = a.dtype if weight is None else _lib.dtype_code(weight.dtype)
    return a


def _forward(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float, keep: bool = False, eight: bool = False):
    """``(out, total, rstd, scale)``: total is x itself without a residual, rstd None unless ``keep``, scale None unless ``eight``."""
    total = x if residual is None else torch.empty_like(residual)
    out = torch.empty(x.shape, dtype=torch.float8_e4m3fn if eight else x.dtype, device=x.device)
    rstd = torch.empty(x.shape[0], dtype=torch.float32, device=x.device) if keep else None
    scale = torch.empty(x.shape[0], dtype=torch.float32, device=x.device) if eight else None
    a = _args(x, weight, total.dtype, eps)
    a.x, a.residual, a.out, a.total = x.data_ptr(), _lib.ptr(residual), out.data_ptr(), total.data_ptr()
    a.rstd, a.scale = _lib.ptr(rstd), _lib.ptr(scale)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib.cgtp_add_rms_forward(C.byref(a), _lib.stream_ptr(x.device)), "cgtp_add_rms_forward")
    return out, total, rstd, scale


def _higher(g_out, inputs, need, g_total, dtype: torch.dtype, eps: float):
    """Gradients of ``(total, weight)`` through the tensor expression of ``out``, of type ``dtype``; what has come in for the total is added."""
    def expression(total, weight):
        t = total.float()
        out = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps)
        if weight is not None:
            out = out * weight.float()
        return out.to(dtype)
    grads = (None, None) if g_out is None else higher_order(expression, inputs, need, g_out)
    if g_total is None or not need[0]:
        return grads
    return g_total if grads[0] is None else grads[0] + g_total, grads[1]


_fallbacks = []


def _fallback(mod):
    """The extension's number for the tensor expression, which a backward under gradient mode evaluates."""
    if not _fallbacks:
        _fallbacks.append(mod.Fallback(_higher))
    return _fallbacks[0]


class _AddRmsNorm(Function):
    """Outputs ``out`` and, with a residual, ``total``: the backward needs neither x nor the residual beside it."""

    @staticmethod
    def forward(ctx, x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float):
        out, total, rstd, _ = _forward(x, residual, weight, eps, True)
        ctx.save_for_backward(total, weight, rstd)
        ctx.eps, ctx.dtype = eps, x.dtype
        ctx.set_materialize_grads(False)
        return out if residual is None else (out, total)

    @staticmethod
    def backward(ctx, g_out, g_total=None):
        total, weight, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        if g_out is None and g_total is None:
            return None, None, None, None
        if torch.is_grad_enabled():
            g, gw = _higher(g_out, (total, weight), (need[0] or need[1], need[2]), g_total, ctx.dtype, ctx.eps)
            return g.to(ctx.dtype) if need[0] else None, g if need[1] else None, gw, None
        same = total.dtype == ctx.dtype                       # then one tensor is the gradient of x and of the residual
        g_out = torch.zeros_like(total, dtype=ctx.dtype) if g_out is None else g_out.contiguous()
        g_total = None if g_total is None else g_total.contiguous()
        a = _args(g_out, weight, total.dtype, ctx.eps)
        a.total, a.rstd, a.grad_out, a.grad_total = total.data_ptr(), rstd.data_ptr(), g_out.data_ptr(), _lib.ptr(g_total)
        gx = torch.empty_like(g_out) if need[0] or (same and need[1]) else None
        gr = gx if same else torch.empty_like(total) if need[1] else None
        gw = torch.empty_like(weight) if need[2] else None
        a.grad_x, a.grad_residual, a.grad_weight = _lib.ptr(gx), 0 if same else _lib.ptr(gr), _lib.ptr(gw)
        nbytes = _lib.lib.cgtp_add_rms_workspace_bytes(C.byref(a))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=total.device) if nbytes else None
        a.workspace = _lib.ptr(ws)
        with torch.cuda.device(total.device):
            _lib.check(_lib.lib.cgtp_add_rms_backward(C.byref(a), _lib.stream_ptr(total.device)), "cgtp_add_rms_backward")
        return gx if need[0] else None, gr if need[1] else None, gw, None


def _checked(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float):
    """The operands as the kernels take them: rows one after the other."""
    _lib.require_gpu(x, residual, weight)
    if x.dtype not in _DTYPES:
        raise CgtpError(f"x must be fp32, bf16 or fp16, got {x.dtype}")
    if residual is not None and x.dtype == torch.float32 and residual.dtype in _DTYPES:
        residual = residual.float()
    for name, t in (("residual", residual), ("weight", weight)):
        if t is None:
            continue
        if t.dtype not in (x.dtype, torch.float32):
            raise CgtpError(f"{name} must be of x's type or fp32, got {t.dtype} with {x.dtype}")
        if t.device != x.device:
            raise CgtpError(f"{name} is on {t.device}, x on {x.device}")
    c = x.shape[-1] if x.ndim else 0
    if not 1 <= c < 1 << 15:
        raise CgtpError(f"x must be (..., C) with 1 <= C < 2^15, got {tuple(x.shape)}")
    if residual is not None and residual.shape != x.shape:
        raise CgtpError(f"residual must have x's shape, got {tuple(residual.shape)} and {tuple(x.shape)}")
    if weight is not None and weight.shape != (c,):
        raise CgtpError(f"weight must be ({c},), got {tuple(weight.shape)}")
    if not (eps == 0.0 or 2.0 ** -126 <= eps <= 2.0 ** 128 * (1 - 2.0 ** -24)):
        raise CgtpError(f"eps must be 0, or above it in fp32's range, got {eps}")
    rows = [None if t is None else t.reshape(-1, c).contiguous() for t in (x, residual)]
    return *rows, None if weight is None else weight.contiguous()


def add_rms_norm(x: Tensor, residual: Optional[Tensor] = None, weight: Optional[Tensor] = None,
                 eps: float = 1e-5) -> Tuple[Tensor, Tensor]:
    """``(out, total)``: ``total = x + residual`` and its root-mean-square norm over the last axis, ``out = total * weight /
    sqrt(mean(total^2) + eps)``.  ``x`` ``(..., C)`` fp32, bf16 or fp16; ``residual`` of x's shape, in its type or in fp32 (16 bits
    beside fp32 are widened); ``weight`` ``(C,)`` likewise.  ``out`` has x's type, ``total`` the residual's, and the norm is that of ``total``
    as it is returned.  Without a residual ``total`` is ``x``.

    Squares and sums are held in 32 bits (elements whose squares leave fp32's range, above 1.8e19, or below 1e-19 where ``eps`` is 0, do not come out as
    their norm; a row of zeros with ``eps`` 0 is NaN); the weight's gradient is summed over the rows in a fixed order.  Differentiable to any order."""
    eps = float(eps)
    keep = (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight))) or _lib.forward_mode()
    flat, flat_residual, w = _checked(x, residual, weight, eps)
    mod = _shim.module()
    if mod is not None:
        out, total = mod.add_rms(flat, flat_residual, w, eps, keep, _fallback(mod))
    elif keep:
        got = _AddRmsNorm.apply(flat, flat_residual, w, eps)
        out, total = (got, None) if residual is None else got
    else:
        out, total = _forward(flat, flat_residual, w, eps)[:2]
    if residual is None:
        return (out if x.ndim == 2 else out.reshape(x.shape)), x
    return (out, total) if x.ndim == 2 else (out.reshape(x.shape), total.reshape(x.shape))


def add_rms_norm_8bit(x: Tensor, residual: Optional[Tensor] = None, weight: Optional[Tensor] = None,
                      eps: float = 1e-5) -> Tuple[Tensor, Tensor, Tensor]:
    """``(values, scale, total)`` of :func:`add_rms_norm` for a product in 8 bits: ``values`` ``(..., C)`` in
    ``torch.float8_e4m3fn`` and ``scale`` ``(...)`` in fp32 with ``out = values * scale[..., None]``, ``scale`` the largest magnitude of the row
    over 448 (0 for a row of zeros, NaN for a row with an infinity or a NaN).  For inference: refused where a gradient would be wanted."""
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight))) or _lib.forward_mode():
        raise CgtpError("an output in 8 bits has no gradient: call under torch.no_grad()")
    eps = float(eps)
    flat, flat_residual, w = _checked(x, residual, weight, eps)
    mod = _shim.module()
    if mod is not None:
        out, scale, total = mod.add_rms_8bit(flat, flat_residual, w, eps)
    else:
        out, total, _, scale = _forward(flat, flat_residual, w, eps, eight=True)
    total = x if residual is None else total.reshape(x.shape)
    return out.reshape(x.shape), scale.reshape(x.shape[:-1]), total
