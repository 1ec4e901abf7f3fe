"""Gradients in gradient mode where autocast is on around the backward: those without it."""
import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("cap", [0.0, 3.0])
def test_expression_of_the_cross_entropy(cap):
    import importlib
    module = importlib.import_module("equitorch_amd.nn.functional.kind_cross_entropy")
    gen = torch.Generator().manual_seed(0)
    x, table = (torch.randn(n, 24, generator=gen).requires_grad_(True) for n in (40, 30))
    kind = torch.randint(-1, 30, (40,), generator=gen)
    want = module._higher(torch.ones(40), (x, table), (True, True), kind, 0.5, cap)
    with torch.autocast("cpu", dtype=BF16):
        got = module._higher(torch.ones(40), (x, table), (True, True), kind, 0.5, cap)
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(got, want))


@pytest.fixture(params=["extension", "ctypes"])
def route(request, monkeypatch):
    from equitorch_amd import _shim
    if request.param == "ctypes":
        monkeypatch.setattr(_shim, "module", lambda: None)
    return request.param


def _both(call, leaves):
    """Gradients with a graph of their own, and those of their squares, without autocast and with it."""
    found = []
    for on in (False, True):
        out = call()
        with torch.autocast("cuda", dtype=BF16, enabled=on):
            grads = torch.autograd.grad(out.sum(), leaves, create_graph=True)
        found.append((*grads, *torch.autograd.grad(sum(g.square().sum() for g in grads), leaves)))
    return found


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_cross_entropy_and_norm(device, route, dtype):
    from equitorch_amd.nn.functional import add_rms_norm, kind_cross_entropy
    x, table = (torch.randn(n, 24, device=device).to(dtype).requires_grad_(True) for n in (40, 30))
    weight, kind = torch.randn(24, device=device).to(dtype).requires_grad_(True), torch.arange(40, device=device) - 10
    want, got = _both(lambda: kind_cross_entropy(x, table, kind, 0.5), (x, table))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    factor = torch.randn(40, 24, device=device)
    want, got = _both(lambda: add_rms_norm(x, None, weight)[0] * factor, (x, weight))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_attention(device, route):
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    plan = AttentionPlan(torch.tensor([0, 7, 20], device=device))
    q, k, v = (torch.randn(20, 2, 16, device=device).requires_grad_(True) for _ in range(3))
    want, got = _both(lambda: segment_attention(q, k, v, plan), (q, k, v))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
