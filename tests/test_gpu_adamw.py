"""The AdamW step over many tensors against its formulas in 64 bits, one step at a time from the states as they were.

Tolerances are bounds on rounding, element by element: half a step of the stored type (a whole one where it is rounded at random),
plus roundings of 2^-24 times the magnitudes that enter."""
import copy

import pytest
import torch

from equitorch_amd import _shim
from equitorch_amd._lib import CgtpError
from equitorch_amd.optim import BLOCK, AdamW
from helpers import stable_seed

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16, E4M3 = torch.float32, torch.float64, torch.bfloat16, torch.float16, torch.float8_e4m3fn
EPS = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -126, BF16: 2.0 ** -126, F16: 2.0 ** -24}
U = 2.0 ** -24


@pytest.fixture(params=["extension", "ctypes"])
def route(request, monkeypatch):
    if request.param == "ctypes":
        monkeypatch.setattr(_shim, "module", lambda: None)
    return request.param


def _within(got, want, bound, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} vs {tuple(want.shape)}"
    excess = ((got - want).abs() - bound).max() if want.numel() else torch.tensor(-1.0)
    assert float(excess) <= 0 and torch.isfinite(got).all(), f"{what}: {float(excess):.3e} over the bound"


def _order(t):
    """The elements in the order of memory."""
    axes = sorted(range(t.ndim), key=lambda i: -t.stride(i))
    return t.detach().permute(axes).reshape(-1).cpu()


def _blocks(flat):
    out = torch.zeros(-(-flat.numel() // BLOCK) * BLOCK, dtype=flat.dtype)
    out[:flat.numel()] = flat
    return out.view(-1, BLOCK)


def _moments(state, bits):
    """(m, v) in 64 bits in the order of memory."""
    if bits == 32:
        return _order(state["exp_avg"]).double(), _order(state["exp_avg_sq"]).double()
    m, r = (_decoded(state, n) for n in ("exp_avg", "root_avg_sq"))
    return m, r.square()


def _decoded(state, name):
    flat = _order(state[name].float()).double()
    return (_blocks(flat) * state[name + "_scale"].cpu().double()[:, None]).view(-1)[:flat.numel()]


def _check_step(opt, group, p, before, grad, weight):
    """One parameter after a step, from its state and weight before it."""
    bits, (b1, b2) = group["state_bits"], group["betas"]
    m, v = _moments(before, bits)
    g = _order(grad).double() * (-1 if group["maximize"] else 1)
    t = float(before["step"]) + 1
    m_size, m, v = b1 * m.abs() + (1 - b1) * g.abs(), b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    lr, decay = float(group["lr"]), group["weight_decay"]
    size, r = lr / (1 - b1 ** t), v.sqrt()
    denominator = r / (1 - b2 ** t) ** 0.5 + group["eps"]
    want = weight * (1 - lr * decay) - size * m / denominator
    # two products and a sum with rounded factors for m (5 roundings), the same for v and half of that in its root; the factors, the
    # products and the quotient
    bound = 3 * U * weight.abs() + size / denominator * (m_size * 5 * U + m.abs() * 16 * U) + 2 * U * want.abs()
    state = opt.state[p]
    assert float(state["step"]) == t
    if "master" in state:
        _within(_order(state["master"]), want, bound, "master")
        assert torch.equal(state["master"].to(p.dtype), p.detach())
    else:
        _within(_order(p), want, bound + EPS[p.dtype] * (want.abs() + bound) + TINY[p.dtype], "p")
    if bits == 32:
        _within(_order(state["exp_avg"]), m, 5 * U * m_size, "exp_avg")
        _within(_order(state["exp_avg_sq"]), v, 6 * U * v + 2.0 ** -126, "exp_avg_sq")
        return
    for name, value, part in (("exp_avg", m, 0.5), ("root_avg_sq", r, 1.0)):
        top = _blocks(value.abs()).amax(1)
        off = 6 * U * (_blocks(m_size).amax(1) if name == "exp_avg" else top)
        _within(state[name + "_scale"], top / 448, off / 448 + 2 * U * top / 448 + 2.0 ** -126, name + "_scale")
        scale = state[name + "_scale"].cpu().double().repeat_interleave(BLOCK)[:value.numel()]
        unit = torch.maximum(2.0 ** (torch.floor(torch.log2((value.abs() / scale.clamp(min=1e-300)).clamp(min=1e-30))) - 3), torch.tensor(2.0 ** -9, dtype=F64))
        slack = (off + 4 * U * top).repeat_interleave(BLOCK)[:value.numel()]
        # where the value lies at a power of two the step above is twice the one below
        _within(_decoded(state, name), value, part * unit * scale * (1 + 2.0 ** -10) + slack, name)
    assert bool((_decoded(state, "root_avg_sq")[r > 0] > 0).all()), "a root above zero became zero"


def _snapshot(opt):
    weights = {}
    for group in opt.param_groups:
        for p in group["params"]:
            weights[p] = _order(opt.state[p].get("master", p)).double() if opt.state[p] else _order(p).double()
    return {p: {k: v.clone() for k, v in s.items()} for p, s in opt.state.items()}, weights


def _fresh(p, bits):
    zero = torch.zeros_like(p, dtype=F32)
    if bits == 32:
        return {"step": torch.zeros(()), "exp_avg": zero, "exp_avg_sq": zero}
    scale = torch.zeros(-(-p.numel() // BLOCK))
    return {"step": torch.zeros(()), "exp_avg": zero, "root_avg_sq": zero, "exp_avg_scale": scale, "root_avg_sq_scale": scale}


def _run(opt, steps, gen, spread=1.0):
    for _ in range(steps):
        for group in opt.param_groups:
            for p in group["params"]:
                size = torch.exp(spread * torch.randn(p.shape, generator=gen))
                p.grad = torch.empty_like(p).copy_(torch.randn(p.shape, generator=gen) * size * 1e-2)
        states, weights = _snapshot(opt)
        opt.step()
        for group in opt.param_groups:
            for p in group["params"]:
                _check_step(opt, group, p, states.get(p) or _fresh(p, group["state_bits"]), p.grad, weights[p])


SHAPES = [(1,), (3,), (255,), (256,), (257,), (64, 4), (33, 31), (5000,), (3, 70, 11), (70001,)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", [(F32, False), (BF16, False), (BF16, True), (F16, True), (F16, False)])
def test_steps(device, route, dtype, master, bits):
    gen = torch.Generator().manual_seed(stable_seed(str(dtype), master, bits))
    params = [torch.nn.Parameter(torch.randn(s, generator=gen).to(device, dtype)) for s in SHAPES]
    _run(AdamW(params, lr=1e-2, weight_decay=0.1, state_bits=bits, master=master, seed=7), 3, gen, 3.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_layouts(device, route, bits):
    """Addresses that are no multiple of 16 bytes, axes in another order, gradients in another order than their parameter."""
    gen = torch.Generator().manual_seed(1)
    flat = torch.randn(4000, generator=gen).to(device)
    params = [flat[1:1025].view(32, 32), flat[1031:1031 + 777], flat[2003:2003 + 600].view(20, 30).T, torch.randn(2, 3, 5, 7, generator=gen).to(device).permute(0, 3, 1, 2),
              torch.randn(40, 50, generator=gen).to(device), torch.zeros((), device=device), torch.zeros(0, 3, device=device),
              torch.randn(6, generator=gen).to(device).as_strided((6, 1, 1), (1, 17, 3))]
    params = [torch.nn.Parameter(p) for p in params]
    assert params[2].data_ptr() == flat.data_ptr() + 4 * 2003
    opt = AdamW(params, lr=1e-2, state_bits=bits)
    for step in range(2):
        for i, p in enumerate(params):
            g = torch.randn(p.shape, generator=gen).to(device)
            p.grad = g.T.contiguous().T if i == 4 else torch.empty_like(p).copy_(g)
        states, weights = _snapshot(opt)
        rest = flat.clone()
        opt.step()
        for p in params:
            grad = torch.empty_like(p).copy_(p.grad)
            _check_step(opt, opt.param_groups[0], p, states.get(p) or _fresh(p, bits), grad, weights[p])
        rest[1:1025], rest[1031:1808], rest[2003:2603] = flat[1:1025], flat[1031:1808], flat[2003:2603]
        assert torch.equal(rest, flat)                   # nothing beside the parameters


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_groups(device, route, bits):
    """More tensors than a launch takes, groups of other numbers and types, parameters without a gradient."""
    gen = torch.Generator().manual_seed(2)
    params = [torch.nn.Parameter(torch.randn(1 + 37 * i % 700, generator=gen).to(device, (F32, BF16)[i % 2])) for i in range(530)]
    opt = AdamW([{"params": params[:500]}, {"params": params[500:], "lr": 3e-2, "betas": (0.0, 0.9), "weight_decay": 0.0, "maximize": True}],
                lr=1e-2, state_bits=bits, seed=11)
    _run(opt, 2, gen)
    idle = params[5]
    kept, count = idle.detach().clone(), float(opt.state[idle]["step"])
    idle.grad = None
    opt.step()
    assert torch.equal(idle, kept) and float(opt.state[idle]["step"]) == count and float(opt.state[params[6]]["step"]) == count + 1


def test_both_routes_are_one(device, monkeypatch):
    """The extension's step and the one through ctypes leave the same bits, in 8 bits too; so do two runs."""
    results = []
    for off in (False, True, False):
        with monkeypatch.context() as patch:
            if off:
                patch.setattr(_shim, "module", lambda: None)
            gen = torch.Generator().manual_seed(3)
            params = [torch.nn.Parameter(torch.randn(n, generator=gen).to(device)) for n in (1000, 77, 30000)]
            opt = AdamW(params, state_bits=8, seed=5)
            for _ in range(4):
                for p in params:
                    p.grad = torch.randn(p.shape, generator=gen).to(device)
                opt.step()
            results.append([p.detach() for p in params] + [opt.state[p][n].float() for p in params for n in ("exp_avg", "root_avg_sq", "root_avg_sq_scale")])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def test_as_torch(device):
    gen = torch.Generator().manual_seed(4)
    start = [torch.randn(s, generator=gen) for s in ((30, 40), (17,))]
    both = []
    for make in (lambda p: AdamW(p, lr=3e-3, weight_decay=0.05), lambda p: torch.optim.AdamW(p, lr=3e-3, weight_decay=0.05)):
        params = [torch.nn.Parameter(t.to(device)) for t in start]
        opt, more = make(params), torch.Generator().manual_seed(5)
        for _ in range(20):
            for p in params:
                p.grad = torch.randn(p.shape, generator=more).to(device)
            opt.step()
        both.append(params)
    for a, b in zip(*both):        # twenty steps of some ten roundings each, of weights below 5
        _within(a, b.detach().cpu(), 20 * 12 * U * 5.0, "p")


def test_eight_bits_follow(device):
    """Rounded at random, a root follows its running mean where to nearest it would never move: the gradients of all elements but
    one a block end, and their roots fall by sqrt(0.999) a step."""
    n = 100 * BLOCK
    p = torch.nn.Parameter(torch.zeros(n, device=device))
    opt = AdamW([p], lr=0.0, state_bits=8, seed=3)
    g = torch.rand(n, generator=torch.Generator().manual_seed(6)).to(device) + 0.5
    p.grad = g
    for _ in range(300):
        opt.step()
    root = lambda: _decoded(opt.state[p], "root_avg_sq").view(-1, BLOCK)                    # noqa: E731
    want = (g.cpu().double() * (1 - 0.999 ** 300) ** 0.5).view(-1, BLOCK)
    # expected: exact but for the concave root (1e-3); an element errs 15 % after some hundred steps, the mean of 25600 0.1 %
    assert abs(float((root() / want).mean()) - 1) < 0.02
    alone = torch.zeros(BLOCK, device=device)
    alone[0] = 2.0
    p.grad, start = alone.repeat(100), root()[:, 1:].mean()
    for _ in range(700):
        opt.step()
    assert abs(float(root()[:, 1:].mean() / start) / 0.999 ** 350 - 1) < 0.02


def test_random_rounding_is_in_proportion(device):
    n = 4000 * BLOCK
    p = torch.nn.Parameter(torch.zeros(n, device=device))
    opt = AdamW([p], betas=(0.9, 0.0), state_bits=8, seed=9)             # v = g^2: the root is |g|
    p.grad = torch.randn(n, generator=torch.Generator().manual_seed(7)).to(device)
    opt.step()
    r = p.grad.abs().cpu().double()
    scale = opt.state[p]["root_avg_sq_scale"].cpu().double().repeat_interleave(BLOCK)
    unit = torch.maximum(2.0 ** (torch.floor(torch.log2(r / scale)) - 3), torch.tensor(2.0 ** -9, dtype=F64)) * scale
    off = (_decoded(opt.state[p], "root_avg_sq") - r) / unit
    keep = r / scale > 2.0 ** -9                                          # below, zero is kept away from
    assert float(off[keep].abs().max()) <= 1.0 + 1e-3
    assert abs(float(off[keep].mean())) <= 5 * 0.5 / n ** 0.5 + 1e-5      # five deviations of a mean of n of at most a half


def test_state_dict(device, tmp_path):
    """Saved and loaded, a run goes on with the same bits, and states keep their types."""
    for bits, dtype, master in ((8, F32, False), (8, BF16, True), (32, BF16, True), (32, F16, False)):
        gen = torch.Generator().manual_seed(8)
        params = [torch.nn.Parameter(torch.randn(s, generator=gen).to(device, dtype)) for s in ((20, 30), (1,), (300,))]
        opt = AdamW(params, lr=1e-2, state_bits=bits, master=master, seed=4)
        grads = [[torch.randn(p.shape, generator=gen).to(device, dtype) for p in params] for _ in range(4)]

        def run(opt, params, grads):
            for gs in grads:
                for p, g in zip(params, gs):
                    p.grad = g
                opt.step()
        run(opt, params, grads[:2])
        torch.save({"p": [p.detach() for p in params], "opt": opt.state_dict()}, tmp_path / "run.pt")
        run(opt, params, grads[2:])
        saved = torch.load(tmp_path / "run.pt", weights_only=True, map_location="cpu")
        others = [torch.nn.Parameter(p.to(device)) for p in saved["p"]]
        again = AdamW(others)
        again.load_state_dict(saved["opt"])
        run(again, others, grads[2:])
        assert again.param_groups[0]["state_bits"] == bits
        for p, q in zip(params, others):
            assert torch.equal(p, q)
            for name, value in opt.state[p].items():
                other = again.state[q][name]
                assert other.dtype == value.dtype and torch.equal(other.float(), value.float()), name


def test_graph_replays(device):
    """A recorded step counts on, follows a learning rate on the GPU, and equals eager steps, which run between the replays."""
    for bits in (32, 8):
        gen = torch.Generator().manual_seed(9)
        start = [torch.randn(s, generator=gen).to(device) for s in ((3000,), (40, 41))]
        sets = [[torch.nn.Parameter(t.clone()) for t in start] for _ in range(2)]
        lrs = [torch.tensor(1e-2, device=device) for _ in range(2)]
        opts = [AdamW(p, lr=lr, state_bits=bits, seed=2) for p, lr in zip(sets, lrs)]
        for params in sets:
            for p in params:
                p.grad = torch.zeros_like(p)

        def fill(seed):
            for params in sets:
                more = torch.Generator().manual_seed(seed)
                for p in params:
                    p.grad.copy_(torch.randn(p.shape, generator=more))
        fill(0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for opt in opts:
                opt.step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opts[0].step()
        for seed in range(1, 5):
            fill(seed)
            for lr in lrs:
                lr.fill_(1e-2 / seed)
            graph.replay()
            torch.cuda.synchronize()
            opts[1].step()
            for p, q in zip(*sets):
                assert torch.equal(p, q) and float(opts[0].state[p]["step"]) == seed + 1
                assert all(torch.equal(opts[0].state[p][n].float(), opts[1].state[q][n].float()) for n in opts[0].state[p])


def test_states_are_not_made_in_a_graph(device):
    p = torch.nn.Parameter(torch.ones(5, device=device))
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(CgtpError):
        with torch.cuda.graph(graph):
            opt.step()
    assert not opt.state[p]
    opt.step()
    assert float(opt.state[p]["step"]) == 1


def test_gradients_that_are_not_finite(device):
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(3 * BLOCK, device=device))
        opt = AdamW([p], state_bits=bits)
        p.grad = torch.ones_like(p)
        p.grad[BLOCK + 5] = float("nan")
        p.grad[2 * BLOCK + 7] = float("inf")
        opt.step()
        assert torch.isnan(p[[BLOCK + 5, 2 * BLOCK + 7]]).all() and int(torch.isnan(p).sum()) == 2
        p.grad = torch.ones_like(p)
        opt.step()
        bad = torch.isnan(p).view(3, BLOCK).sum(1).tolist()
        assert bad == ([0, 1, 1] if bits == 32 else [0, BLOCK, BLOCK])     # in 8 bits a block has one scale


def test_a_step_between_forward_and_backward_is_noticed(device, route):
    p = torch.nn.Parameter(torch.ones(5, device=device))
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    opt.step()
    loss = p.square().sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_closure_and_scaler(device):
    p = torch.nn.Parameter(torch.full((4,), 2.0, device=device))
    opt = AdamW([p], lr=0.1)

    def closure():
        opt.zero_grad()
        loss = p.square().sum()
        loss.backward()
        return loss
    assert float(opt.step(closure).detach()) == 16.0 and float(p.detach()[0]) < 2.0
    scaler, kept = torch.amp.GradScaler("cuda"), None
    for bad in (False, True):
        opt.zero_grad()
        scaler.scale(p.square().sum() * (float("inf") if bad else 1.0)).backward()
        kept = p.detach().clone()
        scaler.step(opt)
        scaler.update()
        assert torch.equal(p, kept) == bad


def test_copies(device):
    p = torch.nn.Parameter(torch.ones(300, device=device))
    opt = AdamW([p], state_bits=8)
    p.grad = torch.ones_like(p)
    opt.step()
    other = copy.deepcopy(opt)
    q = other.param_groups[0]["params"][0]
    q.grad = torch.ones_like(q)
    p.grad = torch.ones_like(p)
    opt.step()
    other.step()
    assert torch.equal(p, q)


def test_refusals(device, route):
    p = torch.nn.Parameter(torch.ones(6, 4, device=device))
    for kwargs in (dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9,)), dict(eps=-1e-8), dict(weight_decay=-0.1),
                   dict(state_bits=16), dict(seed=-1), dict(lr=torch.ones(2, device=device)), dict(lr=torch.ones((), device=device, dtype=F64))):
        with pytest.raises(ValueError):
            AdamW([p], **kwargs)
    base = torch.zeros(20, device=device)
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(base[:12]), torch.nn.Parameter(base[8:])])
    with pytest.raises(ValueError):
        AdamW([p, torch.nn.Parameter(p.detach())])
    opt = AdamW([p])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(p.detach()[2:])]})
    assert len(opt.param_groups) == 1
    for bad in (torch.zeros(3), torch.zeros(3, device=device, dtype=F64), torch.zeros(4, 4, device=device)[:, ::2], torch.zeros(1, device=device).expand(5)):
        q = torch.nn.Parameter(bad)
        q.grad = torch.zeros_like(q)
        with pytest.raises(CgtpError):
            AdamW([q]).step()
    q = torch.nn.Parameter(torch.zeros(4, 3, device=device))
    q.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1, 3), (4, 3)).to(device)
    with pytest.raises(CgtpError):
        AdamW([q]).step()
    p.grad = torch.ones_like(p)
    opt.step()
    for name, value in (("exp_avg", torch.zeros(24, device=device)), ("exp_avg_sq", torch.zeros(6, 4, device=device, dtype=F16)),
                        ("step", torch.zeros(())), ("exp_avg", torch.zeros(4, 6, device=device).T)):
        kept = opt.state[p][name]
        opt.state[p][name] = value
        before = p.detach().clone()
        with pytest.raises(CgtpError):
            opt.step()
        assert torch.equal(p, before)
        opt.state[p][name] = kept
    opt.param_groups[0]["state_bits"] = 8
    with pytest.raises(CgtpError):
        opt.step()


def test_options_changed_later_are_checked(device, route):
    """A number that a schedule or a user sets after the optimizer was made is looked at by the step, before any group's is taken."""
    first, second = (torch.nn.Parameter(torch.ones(6, 4, device=device)) for _ in range(2))
    opt = AdamW([{"params": [first]}, {"params": [second]}])
    first.grad, second.grad = torch.ones_like(first), torch.ones_like(second)
    opt.step()
    group = opt.param_groups[1]
    for name, value in (("lr", -1.0), ("lr", float("nan")), ("lr", torch.ones((), device=device, dtype=F64)), ("lr", torch.ones(2, device=device)),
                        ("betas", (1.0, 0.9)), ("eps", -1e-8), ("weight_decay", float("inf")), ("state_bits", 4), ("seed", 1 << 32)):
        kept, before = group[name], [p.detach().clone() for p in (first, second)]
        group[name] = value
        with pytest.raises(ValueError):
            opt.step()
        group[name] = kept
        assert torch.equal(first, before[0]) and torch.equal(second, before[1])
    group["lr"] = torch.full((), 1e-3, device=device)
    opt.step()
    assert not torch.equal(second, before[1])


def test_the_largest_tensor(device):
    """The end of a tensor whose offsets in bytes pass 32 bits, against the same elements as a tensor of their own."""
    n, tail = (1 << 31) - 100, 256 * 20 + 156      # whole blocks of 256 before the tail, which ends inside one
    assert (n - tail) % 256 == 0
    gen = torch.Generator(device=device).manual_seed(3)
    for bits in (8, 32):
        large = torch.nn.Parameter(torch.zeros(n, device=device, dtype=BF16))
        large.grad = torch.zeros_like(large)
        small = torch.nn.Parameter(torch.randn(tail, device=device, generator=gen).to(BF16))
        small.grad = torch.randn(tail, device=device, generator=gen).to(BF16)
        with torch.no_grad():
            large[n - tail:] = small
            large.grad[n - tail:] = small.grad
        opts = [AdamW([p], lr=1e-1, state_bits=bits) for p in (large, small)]
        for opt in opts:
            opt.step()
        assert torch.equal(large[n - tail:], small) and not large[:n - tail].any()
        a, b = (opt.state[p] for opt, p in zip(opts, (large, small)))
        for name in b:
            if name == "root_avg_sq":
                continue                             # rounded at random by the element's place
            assert torch.equal(a[name].reshape(-1)[-b[name].numel():].float(), b[name].reshape(-1).float()), name


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_eight_bit_states_are_those_of_elementary_operations(device, dtype):
    """Every step's states, bit for bit, by the formulas in operations of 32 bits, each rounded once; roots of 2^-6 and more in units
    of their scale, below which the random bits are added at another place."""
    n, seed, number, (b1, b2) = 256 * 500, 77, 1, (0.9, 0.99)
    gen = torch.Generator().manual_seed(4)
    other, p = (torch.nn.Parameter(torch.randn(k, generator=gen).to(device, dtype)) for k in (5, n))
    opt = AdamW([other, p], lr=1e-3, betas=(b1, b2), state_bits=8, seed=seed)
    m = v = torch.zeros(500, 256, device=device)

    def mixed(h):
        h = (h ^ (h >> 16)) * 0x9C8F2D35 & 0xFFFFFFFF
        h = (h ^ (h >> 15)) * 0xB5297A4D & 0xFFFFFFFF
        return h ^ (h >> 16)

    def scales(x):
        scale = (x.abs().amax(1) * (1 / 448)).clamp(min=2.0 ** -126)
        return scale, (1.0 / scale)[:, None]
    element = torch.arange(n, device=device).view(500, 256)
    for step in range(1, 6):
        g = torch.randn(n, generator=gen).mul(torch.rand(n, generator=gen) + 0.1).to(device, dtype)
        p.grad = g
        opt.step()
        g = g.float().view(500, 256)
        m, v = m * b1 + g * (1 - b1), v * b2 + g * g * (1 - b2)
        state = opt.state[p]
        scale, inverse = scales(m)
        codes = (m * inverse).clamp(-448, 448).to(torch.float8_e4m3fn)
        assert torch.equal(state["exp_avg_scale"], scale) and torch.equal(state["exp_avg"].view(500, 256).view(torch.uint8), codes.view(torch.uint8))
        m = codes.float() * scale[:, None]
        r = v.sqrt()
        scale, inverse = scales(r)
        q = (r * inverse).clamp(max=448.0)
        key = mixed(torch.tensor(seed * 0x85157AF5 + number * 0x9E3779B1 + step * 0xC2B2AE63, device=device) & 0xFFFFFFFF)
        bits = (mixed((key + element * 0x9E3779B1) & 0xFFFFFFFF) >> 12).int()
        want = ((q.view(torch.int32) + bits) & -(1 << 20)).view(torch.float32)
        got = state["root_avg_sq"].view(500, 256).float()
        normal = q >= 2.0 ** -6
        assert torch.equal(state["root_avg_sq_scale"], scale) and torch.equal(got[normal], want[normal]) and normal.float().mean() > 0.99
        v = (got * scale[:, None]).square()
