"""Runs that go on from a saved state on the GPU."""
import copy

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


@pytest.mark.parametrize("bits", [32, 8])
def test_a_recorded_step_goes_on_from_what_was_loaded(device, bits):
    """Back to a saved state between two replays: weights, states, steps and the learning rate on the GPU are those of an eager run."""
    gen = torch.Generator().manual_seed(4)
    start = [torch.randn(s, generator=gen).to(device) for s in ((500,), (30, 41))]
    grads = [[torch.randn(t.shape, generator=gen).to(device) for t in start] for _ in range(6)]

    def make():
        params = [torch.nn.Parameter(t.clone()) for t in start]
        for p in params:
            p.grad = torch.zeros_like(p)
        return params, AdamW(params, lr=torch.full((), 1e-2, device=device), state_bits=bits, seed=3)

    def fill(params, gs):
        for p, g in zip(params, gs):
            p.grad.copy_(g)
    params, opt = make()
    fill(params, grads[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    saved = copy.deepcopy(opt.state_dict())
    weights = [p.detach().clone() for p in params]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for lr in (1e-2, 3e-3):
        for gs in grads[1:4]:
            fill(params, gs)
            graph.replay()
        torch.cuda.synchronize()
        saved["param_groups"][0]["lr"] = lr if lr == 3e-3 else torch.tensor(lr)
        opt.load_state_dict(saved)
        with torch.no_grad():
            for p, w in zip(params, weights):
                p.copy_(w)
        others, eager = make()
        eager.load_state_dict(saved)
        with torch.no_grad():
            for p, w in zip(others, weights):
                p.copy_(w)
        assert eager.param_groups[0]["lr"].is_cuda and float(opt.param_groups[0]["lr"]) == pytest.approx(lr)
        noise = [torch.full((1000,), float("nan"), device=device) for _ in range(50)]      # what is freed is taken
        for gs in grads[4:]:
            fill(params, gs)
            fill(others, gs)
            graph.replay()
            eager.step()
        torch.cuda.synchronize()
        for p, q in zip(params, others):
            assert torch.equal(p, q)
            for name, value in eager.state[q].items():
                assert torch.equal(opt.state[p][name].float(), value.float()), name
        del noise


def test_a_learning_rate_that_groups_share(device):
    """Loaded as one it stays one tensor; loaded as two each group has its own."""
    params = [torch.nn.Parameter(torch.ones(4, device=device)) for _ in range(2)]
    lr = torch.full((), 0.5, device=device)
    opt = AdamW([{"params": [p]} for p in params], lr=lr)
    saved = copy.deepcopy(opt.state_dict())
    lr.fill_(0.1)
    opt.load_state_dict(saved)
    assert all(g["lr"] is lr for g in opt.param_groups) and float(lr) == 0.5
    saved["param_groups"][1]["lr"] = 0.25
    opt.load_state_dict(saved)
    assert [float(g["lr"]) for g in opt.param_groups] == [0.5, 0.25]
