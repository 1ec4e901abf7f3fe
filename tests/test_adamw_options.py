"""Checks of AdamW's options and parameters without a GPU."""
import copy

import pytest
import torch

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
