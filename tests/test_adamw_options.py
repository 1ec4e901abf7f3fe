"""Checks of AdamW's options and parameters without a GPU."""
import copy
import ctypes as C

import pytest
import torch

from equitorch_amd import _lib
from equitorch_amd._lib import AdamwArgs
from equitorch_amd.optim import AdamW


def _params(n=1):
    return [torch.nn.Parameter(torch.zeros(3)) for _ in range(n)]


@pytest.mark.parametrize("value", [-1.0, float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("shape", [(), (1,)])
def test_a_learning_rate_in_a_host_tensor_is_looked_at(value, dtype, shape):
    """By the constructor, by a step, which refuses it before any group is stepped, and by a load."""
    bad = torch.full(shape, value, dtype=dtype)
    with pytest.raises(ValueError):
        AdamW(_params(), lr=bad)
    opt = AdamW([{"params": _params()}, {"params": _params()}], lr=torch.full(shape, 0.1, dtype=dtype))
    opt.step()                                     # no parameter has a gradient
    opt.param_groups[1]["lr"].copy_(bad)
    with pytest.raises(ValueError):
        opt.step()
    saved = AdamW(_params()).state_dict()
    saved["param_groups"][0]["lr"] = bad
    with pytest.raises(ValueError):
        AdamW(_params()).load_state_dict(saved)


def _view(base, begin, end):
    return torch.nn.Parameter(base[begin:end])


def test_overlaps_are_found_whatever_the_groups():
    base = torch.zeros(40)
    parts = [(0, 12), (20, 30), (12, 20)]
    for groups in (lambda: [_view(base, *x) for x in parts], lambda: [{"params": [_view(base, *x)]} for x in parts]):
        assert len(AdamW(groups()).param_groups) in (1, 3)
    for more in ((5, 6), (29, 31), (11, 21)):
        for groups in (lambda: [_view(base, *x) for x in (*parts, more)], lambda: [{"params": [_view(base, *x)]} for x in (*parts, more)]):
            with pytest.raises(ValueError):
                AdamW(groups())
        opt = AdamW([{"params": [_view(base, *x)]} for x in parts])
        for made in (opt, copy.deepcopy(opt)):
            first = made.param_groups[0]["params"][0]
            with pytest.raises(ValueError):
                made.add_param_group({"params": [torch.nn.Parameter(first.detach()[3:5])]})
            assert len(made.param_groups) == 3
    opt.add_param_group({"params": [_view(base, 30, 40)]})
    assert len(opt.param_groups) == 4


def test_construction_looks_at_each_parameter_once(monkeypatch):
    """Of many groups too: the test for overlaps is of all of them together."""
    seen = []
    monkeypatch.setattr(AdamW, "_check_overlap", lambda self: seen.append(len(self.param_groups)))
    opt = AdamW([{"params": [p]} for p in _params(50)])
    assert seen == [50]
    opt.add_param_group({"params": _params()})
    assert seen == [50, 51]


# 1e-50 was zero in 32 bits and 1e-40 had no finite inverse: elements without a gradient became NaN; 1e39 was infinity
@pytest.mark.parametrize("eps,taken", [(1e-50, False), (1e-40, False), (1e39, False), (float("nan"), False), (-1e-8, False), (0.0, True),
                                       (2.0 ** -126, True), (1e-8, True), (3.4e38, True)])
def test_an_eps_that_32_bits_do_not_hold_is_refused(eps, taken):
    a = AdamwArgs()
    a.n_tensors, a.beta1, a.beta2, a.state_bits, a.eps = 0, 0.9, 0.999, 32, eps
    assert _lib.lib.cgtp_adamw_step(C.byref(a), None) == (0 if taken else 5)
    if taken:
        AdamW(_params(), eps=eps).step()
        return
    with pytest.raises(ValueError):
        AdamW(_params(), eps=eps)
    opt = AdamW(_params())
    opt.param_groups[0]["eps"] = eps
    with pytest.raises(ValueError):
        opt.step()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_the_smallest_eps(device, bits):
    """Elements without a gradient stay where they are; one with a gradient takes a step of lr, whatever its size."""
    p = torch.nn.Parameter(torch.ones(600, device=device))
    p.grad = torch.zeros_like(p)
    p.grad[5] = 1e-12
    AdamW([p], lr=0.125, eps=2.0 ** -126, weight_decay=0.0, state_bits=bits).step()
    want = torch.ones(600, dtype=torch.float64, device=device)
    want[5] = 0.875
    # m / sqrt(v) of a first step is 1 to some twelve roundings, of a step of 0.125
    assert bool(((p.detach().double() - want).abs() <= 2.0 ** -24 * (12 * 0.125 + 1)).all())
