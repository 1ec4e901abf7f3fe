"""Checks of AdamW's options and parameters without a GPU."""
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
