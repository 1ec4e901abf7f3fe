"""The norm after a residual's addition against plain implementations in 64 bits on the CPU.

Tolerances are bounds on rounding, element by element: half a step of the result's type, plus the roundings of what is
held in 32 bits times the magnitudes that enter the element."""
import pytest
import torch

from equitorch_amd._lib import CgtpError
from helpers import stable_seed

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
EPS = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -126, BF16: 2.0 ** -126, F16: 2.0 ** -24}


def _rand(gen, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=gen, dtype=F64) * std).to(dtype)


def _within(got, want, bound, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} vs {tuple(want.shape)}"
    excess = ((got - want).abs() - bound).max() if want.numel() else torch.tensor(-1.0)
    assert float(excess) <= 0 and torch.isfinite(got).all(), f"{what}: {float(excess):.3e} over the bound"


def _reference(x, residual, weight, eps):
    """(t, r, out) in 64 bits; t as it is stored."""
    t = x.double() if residual is None else (x.double() + residual.double()).to(residual.dtype).double()
    r = (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    return t, r, t * r * (1.0 if weight is None else weight.double())


TYPES = [(F32, F32, F32), (BF16, BF16, F32), (BF16, F32, BF16), (F16, F16, F16), (F16, F32, F32), (F32, None, None), (BF16, None, F32)]


@pytest.mark.parametrize("dtype,residual_type,weight_type", TYPES)
@pytest.mark.parametrize("rows,channels", [(1, 1), (3, 7), (1000, 8), (257, 9), (30, 64), (5000, 100), (70, 256), (33, 513), (20, 1001),
                                           (3, 2049), (9, 4096), (5, 4097), (2, 16391), (3, 32767), (20000, 40), (1500, 1025), (7, 1995), (6, 6001),
                                           (3, 8200)])
def test_add_rms_norm(device, dtype, residual_type, weight_type, rows, channels):
    from equitorch_amd.nn.functional import add_rms_norm
    gen = torch.Generator().manual_seed(stable_seed(rows, channels, str(dtype)))
    eps = 1e-5
    x = _rand(gen, rows, channels, dtype=dtype)
    residual = None if residual_type is None else _rand(gen, rows, channels, dtype=residual_type, std=2.0)
    weight = None if weight_type is None else _rand(gen, channels, dtype=weight_type)
    total_type = dtype if residual is None else residual_type
    g, gt = _rand(gen, rows, channels, dtype=dtype), _rand(gen, rows, channels, dtype=total_type)
    leaves = [None if v is None else v.to(device).requires_grad_(True) for v in (x, residual, weight)]
    present = [v for v in leaves if v is not None]
    outs = add_rms_norm(*leaves, eps=eps)
    assert outs[0].dtype == dtype and outs[1].dtype == total_type
    grads = iter(torch.autograd.grad(outs, present, (g.to(device), gt.to(device))))
    t, r, out = _reference(x, residual, weight, eps)
    u32 = EPS[F32]
    # a sum of squares in chains of at most 64 (a lane's eight times eight chunks) and 14 more (lanes, wavefronts), the mean and eps:
    # half of these 80 roundings in r; the root errs 2, two products
    _within(outs[1], t, 0.0 * t.abs(), "total")
    stat = (40 + 2 + 2) * u32
    _within(outs[0], out, (EPS[dtype] + stat) * out.abs() + TINY[dtype], "out")
    w = torch.ones(channels, dtype=F64) if weight is None else weight.double()
    g, gt = g.double(), gt.double()
    u, n = g * w, t * r
    grad = gt + r * (u - n * (u * n).mean(-1, keepdim=True))
    size = gt.abs() + r * (u.abs() + n.abs() * (u * n).abs().mean(-1, keepdim=True))
    for name, leaf in (("x", x), ("residual", residual)):
        if leaf is not None:
            # without a residual the two gradients are added after they are rounded
            twice = EPS[dtype] * (size + gt.abs()) if residual is None else 0.0
            _within(next(grads), grad, EPS[leaf.dtype] * grad.abs() + 3 * stat * size + twice + TINY[leaf.dtype], "grad_" + name)
    if weight is not None:
        terms = g * n
        # rows in turn, at most ceil(rows / 1024) of a lane or 32 a workgroup, then lanes, wavefronts and workgroups
        chain = rows / 1024 + 6 + 4 + 32 + 32 + 40
        _within(next(grads), terms.sum(0), EPS[weight_type] * terms.sum(0).abs() + (chain + 44) * u32 * terms.abs().sum(0) + TINY[weight_type],
                "grad_weight")


@pytest.mark.parametrize("rows,channels", [(1, 1), (300, 12), (2000, 256), (20, 1003), (2, 5000)])
@pytest.mark.parametrize("dtype,residual_type", [(F32, F32), (BF16, F32), (F16, None)])
def test_eight_bits(device, dtype, residual_type, rows, channels):
    from equitorch_amd.nn.functional import add_rms_norm_8bit
    gen = torch.Generator().manual_seed(stable_seed(rows, channels))
    x = _rand(gen, rows, channels, dtype=dtype)
    x[0] = 0
    residual = None if residual_type is None else _rand(gen, rows, channels, dtype=residual_type)
    if residual is not None:
        residual[0] = 0
    weight = _rand(gen, channels)
    values, scale, total = add_rms_norm_8bit(x.to(device), None if residual is None else residual.to(device), weight.to(device))
    assert values.dtype == torch.float8_e4m3fn and values.shape == x.shape and scale.shape == (rows,) and scale.dtype == F32
    t, _, out = _reference(x, residual, weight, 1e-5)
    _within(total, t, 0.0 * t.abs(), "total")
    top = out.abs().amax(-1)
    stat = (44 + 3) * EPS[F32]           # as above, and the division, the inverse and the product with it
    _within(scale, top / 448, stat * top / 448, "scale")
    assert float(scale[0]) == 0 and float(values[0].float().abs().max()) == 0
    s = scale.cpu().double()[:, None]
    # half a step of three mantissa bits, or half of the smallest step 2^-9
    bound = torch.maximum(out.abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + stat) + stat * out.abs()
    _within(values.float().cpu().double() * s, out, bound, "values")


def test_eight_bits_of_odd_rows(device):
    """Rows with infinities and NaN, and rows so small that the inverse of the scale would be infinite."""
    from equitorch_amd.nn.functional import add_rms_norm_8bit
    x = torch.randn(5, 70, device=device)
    x[1, 3], x[2, 69] = float("inf"), float("nan")
    x[4] *= 2.0 ** -140 / 16
    values, scale, _ = add_rms_norm_8bit(x, eps=1.0)
    assert torch.isnan(scale[1:3]).all() and torch.isfinite(scale[[0, 3, 4]]).all()
    assert torch.isfinite(values[[0, 3, 4]].float()).all()
    plain = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1.0)
    got = values.float() * scale[:, None]
    assert float((got - plain)[[0, 3]].abs().max()) <= 2.0 ** -4 * float(plain[[0, 3]].abs().max())
    assert float((got - plain)[4].abs().max()) <= 2.0 ** -126


def test_shapes_strides_and_streams(device):
    from equitorch_amd.nn.functional import add_rms_norm
    gen = torch.Generator().manual_seed(3)
    base, res = _rand(gen, 6, 50, 33).to(device), _rand(gen, 50, 33).to(device)
    weight = _rand(gen, 33).to(device)
    x = base[2].T.contiguous().T                       # columns one after the other
    want = add_rms_norm(base[2].contiguous(), res, weight)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = add_rms_norm(x, res, weight)
    torch.cuda.current_stream().wait_stream(side)
    loose = torch.empty(50 * 33 + 1, device=device)[1:].view(50, 33).copy_(base[2])
    for a, b, c in zip(want, got, add_rms_norm(loose, res, weight)):
        assert torch.equal(a, b) and torch.equal(a, c)
    out, total = add_rms_norm(base, None, weight)
    assert out.shape == base.shape and total is base
    out, total = add_rms_norm(base[0, 0], base[1, 0])
    assert out.shape == total.shape == (33,)
    for a in add_rms_norm(base[:0], base[:0], weight):
        assert a.shape == (0, 50, 33)
    leaf = weight.clone().requires_grad_(True)
    (gw,) = torch.autograd.grad(add_rms_norm(base[:0], base[:0], leaf)[0].sum(), leaf)
    assert torch.equal(gw, torch.zeros_like(gw))


def test_one_operand_twice_and_one_output(device):
    """x and the residual are one tensor; only one of the outputs is used."""
    from equitorch_amd.nn.functional import add_rms_norm
    gen = torch.Generator().manual_seed(4)
    x64, w64, g64 = (torch.randn(*s, generator=gen, dtype=F64) for s in ((40, 24), (24,), (40, 24)))
    for which in (0, 1):
        x, w = (v.float().to(device).requires_grad_(True) for v in (x64, w64))
        outs = add_rms_norm(x, x, w)
        gx, gw = torch.autograd.grad(outs[which], (x, w), g64.float().to(device), allow_unused=True)
        a, b = (v.float().double().requires_grad_(True) for v in (x64, w64))
        t = a + a
        out = (t * (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * b, t)[which]
        ga, gb = torch.autograd.grad(out, (a, b), g64.float().double(), allow_unused=True)
        _within(gx, ga, 2e-5 * ga.abs().max(), "x")
        if which == 0:
            _within(gw, gb, 2e-5 * gb.abs().max(), "weight")
        else:
            assert gw is None or torch.equal(gw, torch.zeros_like(gw))


def test_higher_order_and_differences(device):
    from equitorch_amd.nn.functional import add_rms_norm
    gen = torch.Generator().manual_seed(5)
    x, r = (_rand(gen, 9, 20).to(device).requires_grad_(True) for _ in range(2))
    w = _rand(gen, 20).to(device).requires_grad_(True)
    a, b = _rand(gen, 9, 20).to(device), _rand(gen, 9, 20).to(device)

    def value(x, r, w):
        out, total = add_rms_norm(x, r, w)
        return (out * a).sum() + (total * b).sum()

    def plain(x, r, w):
        t = x + r
        return (t * (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * w * a.cpu().double()).sum() + (t * b.cpu().double()).sum()
    got = torch.autograd.grad(value(x, r, w), (x, r, w), create_graph=True)
    twice = torch.autograd.grad(sum(g.square().sum() for g in got), (x, r, w))
    wide = [v.detach().cpu().double().requires_grad_(True) for v in (x, r, w)]
    want = torch.autograd.grad(plain(*wide), wide, create_graph=True)
    more = torch.autograd.grad(sum(g.square().sum() for g in want), wide)
    for p, q in zip((*got, *twice), (*want, *more)):
        _within(p, q.detach(), 1e-4 * q.abs().max(), "gradient")
    # against differences of the kernel's own values: fp32 values err 1e-6 of their size, over a step of 1e-2
    grads = torch.autograd.grad(value(x, r, w), (x, r, w))
    for i, leaf in enumerate((x, r, w)):
        v = _rand(gen, *leaf.shape).to(device)
        ends = [value(*[t.detach() + (s * 1e-2 * v if j == i else 0) for j, t in enumerate((x, r, w))]).double() for s in (1, -1)]
        along = float((grads[i] * v).sum())
        assert abs(float(ends[0] - ends[1]) / 2e-2 - along) <= 2e-2 * (1 + abs(along))


def test_weight_alone(device):
    """Only the weight needs a gradient, with a gradient of the total coming in; in gradient mode too."""
    from equitorch_amd.nn.functional import add_rms_norm
    x, r = torch.randn(11, 16, device=device), torch.randn(11, 16, device=device)
    w = torch.randn(16, device=device, requires_grad=True)
    out, total = add_rms_norm(x, r, w)
    want = (out.detach() / w.detach()).sum(0)
    for create in (False, True):
        (gw,) = torch.autograd.grad(out.sum() + total.sum(), w, create_graph=create, retain_graph=True)
        assert float((gw - want).detach().abs().max()) <= 1e-4 * float(want.abs().max())


def test_graph_replays(device):
    from equitorch_amd.nn.functional import add_rms_norm, add_rms_norm_8bit
    x, r = torch.randn(700, 96, device=device, dtype=BF16, requires_grad=True), torch.randn(700, 96, device=device, requires_grad=True)
    w = torch.randn(96, device=device, requires_grad=True)
    ct = torch.randn(700, 96, device=device, dtype=BF16)

    def step():
        out, total = add_rms_norm(x, r, w)
        with torch.no_grad():
            eight = add_rms_norm_8bit(x, r, w)
        return (out, total, *torch.autograd.grad(out, (x, r, w), ct), eight[0].float(), eight[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for seed in range(3):
        torch.manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(700, 96, device=device))
            r.copy_(torch.randn(700, 96, device=device))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_refusals(device):
    from equitorch_amd.nn.functional import add_rms_norm, add_rms_norm_8bit
    x, w = torch.zeros(3, 8, device=device), torch.ones(8, device=device)
    for bad in ((x.double(),), (x.long(),), (x, x[:2]), (x, x.double()), (x.half(), x.bfloat16()), (x, None, w[:4]), (x, None, w.bfloat16()),
                (x, None, w[None]), (x.cpu(),), (x, x.cpu()), (x[:, :0],), (torch.zeros((), device=device),), (torch.zeros(1, 1 << 15, device=device),)):
        with pytest.raises(CgtpError):
            add_rms_norm(*bad)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(CgtpError):
            add_rms_norm(x, eps=eps)
    with pytest.raises(CgtpError):
        add_rms_norm_8bit(x.requires_grad_(True))
    with torch.no_grad():
        add_rms_norm_8bit(x)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        add_rms_norm(fwd.make_dual(x.detach(), torch.ones_like(x)))


def test_layer(device):
    from equitorch_amd import nn as en
    m = en.AddRMSNorm(30).to(device)
    x, r = torch.randn(4, 7, 30, device=device, dtype=BF16), torch.randn(4, 7, 30, device=device)
    out, total = m(x, r)
    assert out.dtype == BF16 and total.dtype == F32
    _within(total, (x.double() + r.double()).cpu(), 2 * EPS[F32] * (x.abs().double() + r.abs().double()).cpu(), "total")
    out.float().sum().backward()
    assert m.weight.grad.shape == (30,) and torch.isfinite(m.weight.grad).all()


def test_batched_gradients_are_refused(device):
    from equitorch_amd.nn.functional import add_rms_norm
    x = torch.randn(5, 8, device=device, requires_grad=True)
    out, _ = add_rms_norm(x, torch.randn(5, 8, device=device))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, x, torch.ones(3, 5, 8, device=device), is_grads_batched=True)


def test_total_is_kept_from_changes(device):
    """The backward reads total: a change of it in place is noticed."""
    from equitorch_amd.nn.functional import add_rms_norm
    x, r = torch.randn(5, 8, device=device, requires_grad=True), torch.randn(5, 8, device=device)
    out, total = add_rms_norm(x, r)
    with torch.no_grad():
        total.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_offsets_beyond_32_bits(device):
    """The last rows of an array of more than 2^31 elements, against the same rows alone; the weight's gradient has terms of those only."""
    from equitorch_amd.nn.functional import add_rms_norm, add_rms_norm_8bit
    n, c, tail = (1 << 24) + 5003, 129, 3000
    gen = torch.Generator(device=device).manual_seed(1)
    x, r = (torch.zeros(n, c, device=device, dtype=torch.bfloat16) for _ in range(2))
    for t in (x, r):
        t[:7] = t[-tail:] = 1.0
        t[-tail:] *= torch.randn(tail, c, device=device, generator=gen).to(t.dtype)
    weight = torch.randn(c, device=device, generator=gen, requires_grad=True)
    g = torch.zeros_like(x)
    g[-tail:] = torch.randn(tail, c, device=device, generator=gen).to(g.dtype)
    results = []
    for rows in (slice(None), slice(n - tail, None)):
        leaf = x[rows].detach().requires_grad_(True)
        out, total = add_rms_norm(leaf, r[rows], weight)
        gx, gw = torch.autograd.grad(out, (leaf, weight), g[rows])
        values, scale, _ = add_rms_norm_8bit(leaf.detach(), r[rows], weight.detach())
        results.append([t.detach()[-tail:].clone() for t in (out, total, gx, values.view(torch.uint8), scale)] + [gw])
        del out, total, gx, values, leaf
    for a, b in zip(*(t[:5] for t in results)):
        assert torch.equal(a, b)
    t = results[1][1].double()
    size = (g[-tail:].double() * t * (t.square().mean(1, keepdim=True) + 1e-6).rsqrt()).abs().sum(0)
    # two sums of the same 3000 terms in other orders: each at most one rounding of the partial sum a term
    assert ((results[0][5] - results[1][5]).abs().double() <= 2 * 3000 * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("n,c", [(70, 9), (50, 77), (40, 1001), (30, 1501), (20, 3003), (9, 9001), (3, 20003)])
def test_total_in_the_residuals_place(device, n, c):
    import ctypes as C
    from equitorch_amd import _lib
    from equitorch_amd.nn.functional import add_rms_norm
    gen = torch.Generator().manual_seed(n)
    for dtype in (torch.float32, torch.bfloat16):
        x, r = (torch.randn(n, c, generator=gen).to(device, dtype) for _ in range(2))
        out, total = add_rms_norm(x, r, eps=1e-6)
        got = torch.empty_like(x)
        a = _lib.AddRmsArgs()
        a.x, a.residual, a.total, a.out = x.data_ptr(), r.data_ptr(), r.data_ptr(), got.data_ptr()
        a.n_rows, a.channels, a.eps = n, c, 1e-6
        a.dtype = a.residual_dtype = a.weight_dtype = _lib.dtype_code(dtype)
        _lib.check(_lib.lib.cgtp_add_rms_forward(C.byref(a), _lib.stream_ptr(x.device)), "cgtp_add_rms_forward")
        assert torch.equal(r, total) and torch.equal(got, out)


@pytest.mark.parametrize("route", ["extension", "ctypes"])
def test_what_a_backward_keeps(device, route, monkeypatch):
    """total and a number for each row: x and the residual may be freed or written over; gradients of either order are those of them as they were."""
    import gc
    from equitorch_amd import _shim
    from equitorch_amd.nn.functional import add_rms_norm
    if route == "ctypes":
        monkeypatch.setattr(_shim, "module", lambda: None)
    n, c = 5000, 256
    for residual_type in (BF16, F32):
        leaf = torch.randn(n, c, device=device, dtype=BF16, requires_grad=True)
        weight = torch.randn(c, device=device, requires_grad=True)
        gc.collect()
        before = torch.cuda.memory_allocated()
        x, r = leaf * 2, (leaf * 3).to(residual_type)
        out, total = add_rms_norm(x, r, weight)
        del x, r
        kept = torch.cuda.memory_allocated() - before
        # out and total, rstd; the products keep nothing of this size, and allocations are whole blocks of 512 bytes
        assert kept <= n * c * (2 + total.element_size()) + 4 * n + 8 * 512
        g = torch.randn_like(out)
        first = torch.autograd.grad(out, (leaf, weight), g, retain_graph=True)
        second = torch.autograd.grad(out, (leaf, weight), g, create_graph=True)
        for a, b in zip(first, second):
            assert float((a - b).detach().abs().max()) <= 4 * 2.0 ** -8 * float(a.abs().max())
        assert torch.autograd.grad(second[0].float().square().sum(), leaf)[0].isfinite().all()
    x, r = (torch.randn(40, 24, device=device, requires_grad=True) for _ in range(2))
    y = x * 1.0
    out, total = add_rms_norm(y, r)
    want = torch.autograd.grad(out.sum() + total.square().sum(), (x, r), retain_graph=True)
    with torch.no_grad():
        y.zero_()
    got = torch.autograd.grad(out.sum() + total.square().sum(), (x, r))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("route", ["extension", "ctypes"])
def test_a_graph_ends_with_its_results(device, route, monkeypatch):
    """The node keeps an output of its own; that must not keep the node: without a collector of cycles nothing is left of a pass."""
    import gc
    from equitorch_amd import _shim
    from equitorch_amd.nn.functional import add_rms_norm
    if route == "ctypes":
        monkeypatch.setattr(_shim, "module", lambda: None)
    x, r = (torch.randn(4096, 256, device=device, requires_grad=True) for _ in range(2))
    gc.collect()
    gc.disable()
    try:
        before = torch.cuda.memory_allocated()
        for backward in (False, True):
            for _ in range(3):
                out, total = add_rms_norm(x, r)
                if backward:
                    torch.autograd.grad(out.sum() + total.sum(), (x, r))
                del out, total
            assert torch.cuda.memory_allocated() == before
    finally:
        gc.enable()
