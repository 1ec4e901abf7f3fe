"""The operators of a training step together, as the example runs them: norm after a residual between attention and feed-forward blocks,
cross entropy against the embedding's table, AdamW over all parameters; against the same formulas in 64 bits."""
import pytest
import torch

from test_gpu_node_modules import _attend, _close, _example, _feed

pytestmark = pytest.mark.gpu
F64 = torch.float64


class _Wide:
    """A module's parameters as 64-bit leaves, under its names."""

    def __init__(self, module):
        self.module = module
        self.__dict__.update({n: p.detach().cpu().double().requires_grad_(True) for n, p in module.named_parameters()})

    def __getattr__(self, name):
        return getattr(self.__dict__["module"], name)


def _loss_in_64_bits(model, loss, data, hidden):
    """The mean loss of the hidden kinds, and the leaves by the model's own parameters."""
    kind, pos, ptr = (t.cpu() for t in data)
    pos, at = pos.double(), ptr.tolist()
    wide = {m: _Wide(m) for m in model.modules() if list(m.parameters(recurse=False))}
    leaf = lambda m, name: wide[m].__dict__[name]                                                        # noqa: E731

    def norm(m, x):
        return x * (x.square().mean(-1, keepdim=True) + m.eps).rsqrt() * leaf(m, "weight")
    table = leaf(model.embedding, "weight")
    shown = kind.masked_fill(hidden.cpu(), -1)
    x = table[shown.clamp(min=0)] * (shown >= 0)[:, None]
    for layer in model.layers:
        x = x + _attend(wide[layer.attention], norm(layer.norm1, x), at, pos)
        x = x + _feed(wide[layer.feed_forward], norm(layer.norm2, x))
    z = norm(model.norm, x)[hidden.cpu()] @ table.T * loss.scale
    value = torch.nn.functional.cross_entropy(z, kind[hidden.cpu()])
    leaves = {p: leaf(m, n) for m in wide for n, p in m.named_parameters(recurse=False)}
    return value, leaves


@pytest.mark.parametrize("layers", [1, 2])
def test_gradients_and_a_step(device, layers):
    from equitorch_amd import nn as en
    from equitorch_amd.optim import AdamW
    ex = _example()
    torch.manual_seed(layers)
    data = ex.make_structures(5, torch.Generator().manual_seed(layers), device)
    model = ex.StructureEnergy(layers=layers).to(device)
    loss = en.KindCrossEntropy(*model.embedding.weight.shape).to(device)
    loss.weight = model.embedding.weight
    hidden = torch.rand(len(data[0]), device=device) < 0.3
    used = [p for n, p in model.named_parameters() if not n.startswith(("query", "readout", "head"))]
    optimizer = AdamW(used, lr=1e-2, weight_decay=0.1)
    value = ex.hidden_kinds_loss(model, loss, data, hidden)
    value.backward()
    want, leaves = _loss_in_64_bits(model, loss, data, hidden)
    grads = torch.autograd.grad(want, [leaves[p] for p in used])
    _close(value.reshape(1), want.detach().reshape(1), 1e-3)
    for p, g in zip(used, grads):
        assert float((p.grad.cpu().double() - g).abs().max()) <= 1e-3 * max(1e-3, float(g.abs().max()))
    before = [p.detach().cpu().double() for p in used]
    optimizer.step()
    for p, w in zip(used, before):
        g = p.grad.cpu().double()
        # the first step: m / (1 - b1) and v / (1 - b2) are g and g^2
        step = w * (1 - 1e-2 * 0.1) - 1e-2 * g / (g.abs() + 1e-8)
        assert float((p.detach().cpu().double() - step).abs().max()) <= 1e-6 * max(1.0, float(step.abs().max()))


def test_example_pretrains(device):
    """Runs, in 32 and with 16-bit blocks; every parameter that is asked for moves and stays finite."""
    ex = _example()
    for half in (False, True):
        torch.manual_seed(3)
        data = ex.make_structures(8, torch.Generator().manual_seed(3), device)
        model = ex.StructureEnergy().to(device)
        if half:
            model.operands(torch.bfloat16)
        before = {n: p.detach().clone() for n, p in model.named_parameters()}
        losses = ex.pretrain(model, data, 3)
        assert losses.shape == (3,) and torch.isfinite(losses).all()
        for n, p in model.named_parameters():
            assert torch.isfinite(p).all()
            assert torch.equal(p, before[n]) == n.startswith(("query", "readout", "head")), n


def test_a_recorded_training_step(device):
    """Norm, loss, backward and optimizer in one graph: replays equal eager steps."""
    from equitorch_amd import nn as en
    from equitorch_amd.optim import AdamW
    runs = []
    x, kind = torch.randn(300, 24, device=device), torch.randint(-1, 40, (300,), device=device)
    for recorded in (False, True):
        torch.manual_seed(4)
        norm, loss, block = en.AddRMSNorm(24).to(device), en.KindCrossEntropy(40, 24).to(device), en.GatedFeedForward(24, 48).to(device)
        params = [p for m in (norm, loss, block) for p in m.parameters()]
        opt = AdamW(params, lr=1e-2, state_bits=8)
        out = torch.zeros((), device=device)

        def step():
            h, total = norm(x)
            update = block(h)
            value = loss(norm(update, total)[0], kind).mean()
            for p, g in zip(params, torch.autograd.grad(value, params)):
                p.grad = g
            opt.step()
            out.copy_(value.detach())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        if recorded:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        values = []
        for _ in range(4):
            graph.replay() if recorded else step()
            torch.cuda.synchronize()
            values.append(float(out))
        runs.append((values, [p.detach().clone() for p in params]))
    assert runs[0][0] == runs[1][0] and all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))


def test_two_graphs_and_two_streams_at_once(device):
    """Calls of different sizes side by side, eager on two streams and as two graphs that share a pool in turn: nothing of one is in another."""
    from equitorch_amd.nn.functional import add_rms_norm, kind_cross_entropy
    sizes = [(3000, 200, 64, torch.bfloat16), (900, 5000, 120, torch.float32)]
    gen = torch.Generator(device=device).manual_seed(8)
    work = []
    for n, k, c, dtype in sizes:
        x, r, table = (torch.randn(m, c, device=device, generator=gen).to(dtype).requires_grad_(True) for m in (n, n, k))
        work.append((x, r, table, torch.randint(-50, k, (n,), device=device, generator=gen), torch.rand(n, device=device, generator=gen)))

    def step(x, r, table, kind, g):
        out, _ = add_rms_norm(x, r)
        loss = kind_cross_entropy(out, table, kind, 0.1)
        # no result holds the autograd graph: one of the same leaves that is alive while a backward is captured ends the capture, and the process
        return [t.detach() for t in (loss, *torch.autograd.grad(loss, (x, r, table), g))]
    want = [step(*w) for w in work]
    streams = [torch.cuda.Stream() for _ in work]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[] for _ in work]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*work[i]))
    torch.cuda.synchronize()
    for results, one in zip(got, want):
        assert all(torch.equal(a, b) for result in results for a, b in zip(result, one))
    del got
    graphs, kept, pool = [], [], None
    for w in work:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            kept.append(step(*w))
        graphs.append(graph)
        pool = graph.pool()
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        step(*work[0])
        torch.cuda.synchronize()
        for results, one in zip(kept, want):
            assert all(torch.equal(a, b) for a, b in zip(results, one))
