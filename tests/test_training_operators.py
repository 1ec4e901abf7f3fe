"""The operators of a training step on invariant channels without a GPU: layouts of the argument structs and the codes of
refused calls."""
import ctypes as C

import pytest
import torch

from equitorch_amd import _lib
from equitorch_amd._lib import AdamwArgs, AdamwTensor, AddRmsArgs, CgtpError, KindLossArgs

NULL, SHAPE, ALIGN, DTYPE, CONFIG, WORKSPACE = 1, 2, 3, 4, 5, 8


@pytest.mark.parametrize("which,cls", [(20, AddRmsArgs), (21, KindLossArgs), (22, AdamwTensor), (23, AdamwArgs)])
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


# ---- cross entropy over kinds ------------------------------------------------------------------------------------
def _loss(**changed):
    a = KindLossArgs()
    for name in ("x", "table", "kind", "loss", "lse", "grad_loss", "grad_x", "grad_table", "workspace"):
        setattr(a, name, 4096)
    a.n_rows, a.n_kinds, a.channels, a.scale = 5, 7, 8, 1.0
    for name, value in changed.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changed,forward,backward", [
    ({"dtype": 1}, DTYPE, DTYPE), ({"channels": 0}, SHAPE, SHAPE), ({"channels": 1 << 15}, SHAPE, SHAPE), ({"n_rows": -1}, SHAPE, SHAPE),
    ({"n_rows": (1 << 29) + 1}, SHAPE, SHAPE), ({"n_kinds": 0}, SHAPE, SHAPE), ({"n_kinds": (1 << 30) + 1}, SHAPE, SHAPE), ({"x": None}, NULL, NULL),
    ({"table": None}, NULL, NULL), ({"kind": None}, NULL, NULL), ({"loss": None}, NULL, None), ({"lse": None}, None, NULL),
    ({"grad_loss": None}, None, NULL), ({"workspace": None}, WORKSPACE, WORKSPACE), ({"workspace": 4104}, ALIGN, ALIGN)])
def test_kind_loss_codes(changed, forward, backward):
    a = _loss(**changed)
    if forward is not None:
        assert _lib.lib.cgtp_kind_loss_forward(C.byref(a), None) == forward
    if backward is not None:
        assert _lib.lib.cgtp_kind_loss_backward(C.byref(a), None) == backward
    assert _lib.lib.cgtp_kind_loss_forward(None, None) == _lib.lib.cgtp_kind_loss_backward(None, None) == NULL


def test_kind_loss_without_work():
    assert _lib.lib.cgtp_kind_loss_forward(C.byref(_loss(n_rows=0, x=None, kind=None, workspace=None)), None) == 0
    assert _lib.lib.cgtp_kind_loss_backward(C.byref(_loss(n_rows=0, grad_table=None)), None) == 0
    assert _lib.lib.cgtp_kind_loss_backward(C.byref(_loss(grad_x=None, grad_table=None)), None) == 0


def test_kind_loss_workspace():
    need = lambda backward, **changed: _lib.lib.cgtp_kind_loss_workspace_bytes(C.byref(_loss(**changed)), backward)
    assert need(0, n_rows=0) == need(1, n_rows=0) == need(1, channels=0) == 0
    large = dict(n_rows=16384, n_kinds=30000, channels=256, dtype=2)
    logits = 2 * 65536 * 60000
    large.update(n_rows=65536, n_kinds=60000)
    assert 2 * 65536 * 256 < need(0, **large) < logits / 16 and need(1, **large) < logits / 6
    assert need(1, **{**large, "grad_table": None}) < need(1, **large)
    # a table whose rows are not whole aligned chunks is copied
    assert need(0, **{**large, "table": 4098}) - need(0, **large) == 2 * 60000 * 256
    # the most rows and kinds there may be: no overflow
    assert need(1, n_rows=1 << 29, n_kinds=1 << 30, channels=(1 << 15) - 1) > 1 << 45


def test_kind_cross_entropy_takes_gpu_tensors_only():
    from equitorch_amd.nn.functional import kind_cross_entropy
    with pytest.raises(CgtpError):
        kind_cross_entropy(torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64))


def test_kind_cross_entropy_layer():
    from equitorch_amd import nn as en
    m = en.KindCrossEntropy(5, 16, cap=3.0)
    assert m.weight.shape == (5, 16) and m.scale == 0.25 and "cap=3.0" in repr(m)
    for make in (lambda: en.KindCrossEntropy(0, 4), lambda: en.KindCrossEntropy(4, 0), lambda: en.KindCrossEntropy(4, 4, cap=0.0)):
        with pytest.raises(ValueError):
            make()


# ---- AdamW ---------------------------------------------------------------------------------------------------------
def _adamw(tensor=None, **changed):
    t = (AdamwTensor * 1)()
    for name in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master", "step"):
        setattr(t[0], name, 4096)
    t[0].n = 10
    for name, value in (tensor or {}).items():
        setattr(t[0], name, value)
    a = AdamwArgs()
    a.tensors, a.n_tensors, a.beta1, a.beta2, a.state_bits = t, 1, 0.9, 0.999, 32
    for name, value in changed.items():
        setattr(a, name, value)
    return a, t


@pytest.mark.parametrize("tensor,changed,status", [
    ({}, {"dtype": 1}, DTYPE), ({}, {"state_bits": 16}, CONFIG), ({}, {"n_tensors": -1}, SHAPE), ({}, {"beta1": 1.0}, CONFIG), ({}, {"beta2": -0.1}, CONFIG),
    ({}, {"beta1": float("nan")}, CONFIG), ({}, {"tensors": None}, NULL), ({"n": -1}, {}, SHAPE), ({"n": 1 << 31}, {}, SHAPE), ({"param": None}, {}, NULL),
    ({"grad": None}, {}, NULL), ({"exp_avg": None}, {}, NULL), ({"exp_avg_sq": None}, {}, NULL), ({"step": None}, {}, NULL),
    ({"exp_avg_scale": None}, {"state_bits": 8}, NULL), ({"exp_avg_sq_scale": None}, {"state_bits": 8}, NULL), ({"master": None}, {"master": 1, "dtype": 2}, NULL),
    ({}, {"master": 1}, CONFIG)])
def test_adamw_codes(tensor, changed, status):
    a, _ = _adamw(tensor, **changed)
    assert _lib.lib.cgtp_adamw_step(C.byref(a), None) == status
    assert _lib.lib.cgtp_adamw_step(None, None) == NULL


def test_adamw_without_work():
    a, _ = _adamw(n_tensors=0, tensors=None)
    assert _lib.lib.cgtp_adamw_step(C.byref(a), None) == 0


def test_adamw_takes_gpu_tensors_only():
    from equitorch_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(CgtpError):
        AdamW([p]).step()
    p.grad = None
    AdamW([p]).step()
    with pytest.raises(ValueError):
        AdamW([p], state_bits=4)
