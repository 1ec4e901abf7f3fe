"""What the norm after a residual keeps between calls."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_one_callable_for_every_eps(device):
    """Gradients of higher order know their own eps, and a program that has many keeps no callable for each."""
    import importlib
    module = importlib.import_module("equitorch_amd.nn.functional.add_rms_norm")
    x, weight = torch.randn(9, 16, device=device, requires_grad=True), torch.randn(16, device=device, requires_grad=True)
    factor = torch.randn(9, 16, device=device)
    outs = {eps: module.add_rms_norm(x, None, weight, eps)[0] for eps in [10.0 ** -i for i in range(8)] + [0.0, 3.0]}
    for eps, out in outs.items():
        got = torch.autograd.grad((out * factor).sum(), (x, weight), create_graph=True)
        wide = [t.detach().double().requires_grad_(True) for t in (x, weight)]
        want = torch.autograd.grad((wide[0] * torch.rsqrt(wide[0].square().mean(-1, keepdim=True) + eps) * wide[1] * factor.double()).sum(), wide)
        for a, b in zip(got, want):
            # sums over 16 channels or nine rows of terms with some twenty roundings, their magnitudes within eight times the largest gradient
            assert bool(((a.double() - b).abs() <= 2.0 ** -24 * 400 * b.abs().max()).all()), eps
    assert len(module._fallbacks) <= 1
