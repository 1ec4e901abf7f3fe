"""The operators of a training step on invariant channels without a GPU: layouts of the argument structs and the codes of
refused calls."""
import ctypes as C

import pytest
import torch

from equitorch_amd import _lib
from equitorch_amd._lib import AddRmsArgs, CgtpError

NULL, SHAPE, ALIGN, DTYPE, CONFIG, WORKSPACE = 1, 2, 3, 4, 5, 8


@pytest.mark.parametrize("which,cls", [(20, AddRmsArgs)])
def test_struct_layouts(which, cls):
    n = _lib.lib.cgtp_abi_layout(which, None, 0)
    assert n == 1 + len(cls._fields_)
    buf = (C.c_int64 * n)()
    assert _lib.lib.cgtp_abi_layout(which, buf, n) == n
    assert list(buf) == [C.sizeof(cls)] + [getattr(cls, name).offset for name, _ in cls._fields_]


# ---- norm after a residual's addition ------------------------------------------------------------------------------
def _rms(**changed):
    a = AddRmsArgs()
    for name in ("x", "residual", "weight", "out", "total", "rstd", "grad_out", "grad_x", "grad_weight", "workspace"):
        setattr(a, name, 4096)
    a.n_rows, a.channels, a.eps = 5, 8, 1e-5
    for name, value in changed.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changed,forward,backward", [
    ({"dtype": 1}, DTYPE, DTYPE), ({"dtype": 2, "residual_dtype": 3, "weight_dtype": 2}, DTYPE, DTYPE), ({"residual_dtype": 2}, DTYPE, DTYPE),
    ({"dtype": 2, "residual_dtype": 2, "weight_dtype": 3}, DTYPE, DTYPE), ({"channels": 0}, SHAPE, SHAPE), ({"channels": 1 << 15}, SHAPE, SHAPE),
    ({"n_rows": -1}, SHAPE, SHAPE), ({"n_rows": 1 << 31}, SHAPE, SHAPE), ({"x": None}, NULL, None), ({"out": None}, NULL, None),
    ({"total": None}, None, NULL), ({"rstd": None}, None, NULL), ({"grad_out": None}, None, NULL)])
def test_add_rms_codes(changed, forward, backward):
    a = _rms(**changed)
    if forward is not None:
        assert _lib.lib.cgtp_add_rms_forward(C.byref(a), None) == forward
    if backward is not None:
        assert _lib.lib.cgtp_add_rms_backward(C.byref(a), None) == backward
    assert _lib.lib.cgtp_add_rms_forward(None, None) == _lib.lib.cgtp_add_rms_backward(None, None) == NULL


def test_add_rms_without_work():
    assert _lib.lib.cgtp_add_rms_forward(C.byref(_rms(n_rows=0, x=None, out=None)), None) == 0
    assert _lib.lib.cgtp_add_rms_backward(C.byref(_rms(grad_x=None, grad_weight=None)), None) == 0


def test_add_rms_workspace():
    need = lambda **changed: _lib.lib.cgtp_add_rms_workspace_bytes(C.byref(_rms(**changed)))
    assert need(n_rows=100000, channels=64) > 0 and need(n_rows=100000, channels=64) % (4 * 64) == 0
    assert need(n_rows=100000, grad_weight=None) == need(n_rows=0) == need(channels=0) == need(n_rows=3) == 0
    assert _lib.lib.cgtp_add_rms_backward(C.byref(_rms(n_rows=100000, channels=64, workspace=None)), None) == WORKSPACE


def test_add_rms_norm_takes_gpu_tensors_only():
    from equitorch_amd.nn.functional import add_rms_norm, add_rms_norm_8bit
    for fn in (add_rms_norm, add_rms_norm_8bit):
        with pytest.raises(CgtpError):
            fn(torch.zeros(3, 4))


def test_add_rms_layer():
    from equitorch_amd import nn as en
    m = en.AddRMSNorm(12, eps=1e-6)
    assert m.weight.shape == (12,) and "channels=12" in repr(m) and en.AddRMSNorm(3, affine=False).weight is None
    for make in (lambda: en.AddRMSNorm(0), lambda: en.AddRMSNorm(4, eps=-1.0), lambda: en.AddRMSNorm(4, eps=float("inf")), lambda: m(torch.zeros(3, 4))):
        with pytest.raises(ValueError):
            make()
