"""Values of eps that 32 bits do not hold are refused: without a GPU, by the codes of the C entries."""
import ctypes as C

import pytest
import torch

from equitorch_amd import _lib
from equitorch_amd._lib import AddRmsArgs, CgtpError

CONFIG = 5
# 1e-46 was zero, and a row of zeros NaN; 1e39 was infinity, and every row zeros
BAD = [1e-46, 1e-39, 1e39, -1e-5, float("nan"), float("inf")]
GOOD = [0.0, 2.0 ** -126, 1e-5, 3.4e38]


def _args(eps):
    a = AddRmsArgs()
    a.n_rows, a.channels, a.eps = 0, 8, eps
    return a


@pytest.mark.parametrize("eps", BAD)
def test_codes_of_what_is_refused(eps):
    a = _args(eps)
    assert _lib.lib.cgtp_add_rms_forward(C.byref(a), None) == CONFIG
    assert _lib.lib.cgtp_add_rms_backward(C.byref(a), None) == CONFIG


@pytest.mark.parametrize("eps", GOOD)
def test_codes_of_what_is_taken(eps):
    a = _args(eps)
    assert _lib.lib.cgtp_add_rms_forward(C.byref(a), None) == 0
    assert _lib.lib.cgtp_add_rms_backward(C.byref(a), None) == 0


@pytest.mark.gpu
def test_refusals_and_extremes(device):
    from equitorch_amd.nn.functional import add_rms_norm, add_rms_norm_8bit
    x = torch.tensor([[0.0] * 5, [1e-3, -2e-3, 0.0, 5e-4, 1e-3]], device=device)
    for eps in BAD:
        for fn in (add_rms_norm, add_rms_norm_8bit):
            with pytest.raises(CgtpError):
                fn(x, None, None, eps)
    for eps in GOOD:
        leaf = x[int(eps == 0):].requires_grad_(True)
        out, _ = add_rms_norm(leaf, None, None, eps)
        wide = leaf.detach().double().requires_grad_(True)
        want = wide / (wide.square().mean(-1, keepdim=True) + eps).sqrt()
        factor = torch.arange(5.0, device=device)
        for a, b in ((out, want), (torch.autograd.grad((out * factor).sum(), leaf)[0], torch.autograd.grad((want * factor).sum(), wide)[0])):
            # fewer than sixty roundings of terms of the size of the row's largest; below the normal numbers a step of them
            assert bool(((a - b).abs() <= 2.0 ** -24 * 60 * b.abs().amax(-1, keepdim=True) + 2.0 ** -148).all()), eps
