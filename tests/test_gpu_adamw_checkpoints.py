"""Runs that go on from a saved state on the GPU."""
import pytest
import torch

from equitorch_amd.optim import AdamW

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def test_goes_on_from_torchs_adamw(device):
    """Steps after three of torch's are those that torch's take in 64 bits from the same numbers."""
    gen = torch.Generator().manual_seed(3)
    shapes, lr, (b1, b2), eps, decay = ((40, 50), (7,), ()), 0.01, (0.9, 0.99), 1e-8, 0.1
    grads = [[torch.randn(s, generator=gen).to(device) for s in shapes] for _ in range(4)]
    first = [torch.nn.Parameter(torch.randn(s, generator=gen).to(device)) for s in shapes]
    theirs = torch.optim.AdamW(first, lr=lr, betas=(b1, b2), eps=eps, weight_decay=decay)
    for gs in grads[:3]:
        for p, g in zip(first, gs):
            p.grad = g
        theirs.step()
    second = [torch.nn.Parameter(p.detach().clone()) for p in first]
    opt = AdamW(second)
    opt.load_state_dict(theirs.state_dict())
    for p, q, g in zip(first, second, grads[3]):
        q.grad = g
        s = theirs.state[p]
        m, v, w = s["exp_avg"].double(), s["exp_avg_sq"].double(), p.detach().double()
        size = b1 * m.abs() + (1 - b1) * g.double().abs()
        m, v = b1 * m + (1 - b1) * g.double(), b2 * v + (1 - b2) * g.double() ** 2
        step, below = lr / (1 - b1 ** 4), (v / (1 - b2 ** 4)).sqrt() + eps
        q.want = w * (1 - lr * decay) - step * m / below
        # the products of the weight and of m with rounded factors, and some sixteen roundings of the quotient
        q.bound = U * (3 * w.abs() + step / below * (5 * size + 16 * m.abs()) + 3 * q.want.abs())
    opt.step()
    for q in second:
        assert bool(((q.detach().double() - q.want).abs() <= q.bound).all())
        assert float(opt.state[q]["step"]) == 4
