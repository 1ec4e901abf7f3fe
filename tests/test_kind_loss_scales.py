"""Scales and caps that the cross entropy's kernels cannot hold in 32 bits are refused: without a GPU, by the codes of the C entries."""
import ctypes as C

import pytest
import torch

from equitorch_amd import _lib
from equitorch_amd._lib import CgtpError, KindLossArgs

CONFIG = 5
# scale / cap below fp32's normal numbers was zero, or had a few bits: the logits were zeros, or off by as much
BAD = [(1e-8, 1e38), (1e-3, 1e38), (-1e-3, 1e38), (1e-39, None), (-1e-44, 2.0), (2.0 ** -100, 2.0 ** 27)]
GOOD = [(1e-8, 1e29), (0.0, 1e38), (0.0, None), (2.0 ** -126, None), (2.0 ** -100, 2.0 ** 26), (1e38, 1.0), (1.0, 8e37), (-0.5, 1e-37)]


def _args(scale, cap):
    a = KindLossArgs()
    a.n_rows, a.n_kinds, a.channels, a.scale, a.cap = 0, 7, 8, scale, cap or 0.0
    return a


@pytest.mark.parametrize("scale,cap", BAD + [(float("nan"), None), (float("inf"), None), (1e38, 0.1), (1.0, 1e-39), (1.0, float("inf")), (1.0, float("nan"))])
def test_codes_of_what_is_refused(scale, cap):
    a = _args(scale, cap)
    assert _lib.lib.cgtp_kind_loss_forward(C.byref(a), None) == CONFIG
    assert _lib.lib.cgtp_kind_loss_backward(C.byref(a), None) == CONFIG
    a.n_rows = 5
    assert _lib.lib.cgtp_kind_loss_workspace_bytes(C.byref(a), 1) == 0


@pytest.mark.parametrize("scale,cap", GOOD)
def test_codes_of_what_is_taken(scale, cap):
    assert _lib.lib.cgtp_kind_loss_forward(C.byref(_args(scale, cap)), None) == 0
    assert _lib.lib.cgtp_kind_loss_backward(C.byref(_args(scale, cap)), None) == 0


@pytest.mark.gpu
def test_refusals_and_extremes(device):
    from equitorch_amd.nn.functional import kind_cross_entropy
    gen = torch.Generator().manual_seed(1)
    x, w = torch.randn(6, 8, generator=gen), torch.randn(7, 8, generator=gen)
    kind = torch.arange(6)
    for scale, cap in BAD:
        with pytest.raises(CgtpError):
            kind_cross_entropy(x.to(device), w.to(device), kind.to(device), scale, cap)
    for scale, cap in GOOD:
        for dtype in (torch.float32, torch.bfloat16):
            a, b = (t.to(dtype).double() for t in (x, w))
            z = a @ b.T * scale
            z = cap * torch.tanh(z / cap) if cap else z
            got = kind_cross_entropy(x.to(device, dtype), w.to(device, dtype), kind.to(device), scale, cap).cpu().double()
            want = torch.logsumexp(z, 1) - z.gather(1, kind[:, None])[:, 0]
            # the product's twelve roundings, ten of the tangent, and those of maximum, sum, logarithm and difference
            most = (a.abs() @ b.abs().T).amax(1) * abs(scale)
            bound = 2.0 ** -24 * (12 * most + (3 * cap if cap and abs(scale) / cap > 1e-3 else 0) + 20 * z.abs().amax(1) + 50)
            assert bool(((got - want).abs() <= bound).all()), (scale, cap, dtype)
