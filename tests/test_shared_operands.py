"""First-order gradients taken in gradient mode (forces in the loss) are the ones taken without it, where one operand of an
operator is, or is computed from, another: queries, keys and values of one tensor, positions, harmonics, angles and weights
that two layers share.  And the force loss's parameter gradients of a whole model against 64 bits."""
import pytest
import torch
from torch.autograd import Function

from equitorch_amd.nn.functional._higher_order import higher_order

gpu = pytest.mark.gpu
F32, F64 = torch.float32, torch.float64


def _rand(gen, *shape, dtype=F64, std=1.0):
    return (torch.randn(*shape, generator=gen, dtype=F64) * std).to(dtype)


def _both_ways(function, leaves, gen, tol, second=True):
    """``tol``: of the largest element of a gradient.  The gradient of the gradient against differences in 64 bits is the other
    tests' matter; here it has to exist."""
    out = function(*leaves)
    ct = torch.randn(out.shape, generator=gen, dtype=F64).to(out)
    plain = torch.autograd.grad(out, leaves, ct, retain_graph=True)
    graph = torch.autograd.grad(out, leaves, ct, create_graph=True)
    for i, (a, b) in enumerate(zip(plain, graph)):
        assert float((a - b.detach()).abs().max()) <= tol * max(1e-3, float(a.abs().max())), f"leaf {i}"
    if second:
        for g in torch.autograd.grad(sum(b.square().sum() for b in graph), leaves, allow_unused=True):
            assert g is None or bool(torch.isfinite(g).all())


def _as_operator(expression, inputs):
    """An operator whose backward in gradient mode is the tensor expression, as the library's are, with the
    gradients otherwise by autograd on copies: it runs on the CPU."""
    class Operator(Function):
        @staticmethod
        def forward(ctx, *t):
            ctx.save_for_backward(*t)
            return expression(*t)

        @staticmethod
        def backward(ctx, g):
            t, need = ctx.saved_tensors, ctx.needs_input_grad
            if torch.is_grad_enabled():
                return higher_order(expression, t, need, g)
            with torch.enable_grad():
                own = [None if x is None else x.detach().requires_grad_(True) for x in t]
                got = torch.autograd.grad(expression(*own), [x for x in own if x is not None], g, allow_unused=True)
            got = iter(got)
            return tuple(None if x is None else next(got) for x in own)
    return Operator.apply(*inputs)


def test_expression_of_inputs_that_depend_on_one_another():
    gen = torch.Generator().manual_seed(1)
    x, w = _rand(gen, 5, 4).requires_grad_(True), _rand(gen, 4, 4).requires_grad_(True)
    product = lambda a, b, c: torch.tanh(a @ b) * c.square()
    _both_ways(lambda x, w: _as_operator(product, (x, w, x)), [x, w], gen, 1e-13)
    _both_ways(lambda x, w: _as_operator(product, (_as_operator(product, (x, w, x)), w, x)), [x, w], gen, 1e-13)
    # the gradient of the gradient, against differences
    layers = lambda x, w: _as_operator(product, (_as_operator(product, (x, w, x)), w, x))
    assert torch.autograd.gradgradcheck(layers, (x, w))
    # what nothing depends on, and what is not there
    got = higher_order(lambda a, b, c: a * 2.0, (x, w, None), (True, True, False), torch.ones_like(x))
    assert torch.equal(got[0], torch.full_like(x, 2.0)) and got[1] is None and got[2] is None


@pytest.mark.parametrize("case", ["one tensor", "keys and values", "layers"])
def test_expression_of_the_attention(case):
    from equitorch_amd.nn.functional import AttentionPlan
    from equitorch_amd.nn.functional.attention import _of_buckets
    gen = torch.Generator().manual_seed(2)
    buckets = AttentionPlan(torch.tensor([0, 5, 5, 12]))._buckets
    attend = lambda *t: _as_operator(_of_buckets(buckets, 0.5, 3.0), t)
    x, pos, slope = (_rand(gen, 12, 2, 4, dtype=F32).requires_grad_(True), _rand(gen, 12, 3, dtype=F32).requires_grad_(True),
                     torch.rand(2, generator=gen).requires_grad_(True))
    function = {"one tensor": lambda x, pos, slope: attend(x, x, x, pos, None, slope),
                "keys and values": lambda x, pos, slope: attend(x, x * 2.0, x * 2.0, pos, pos, slope),
                "layers": lambda x, pos, slope: attend(*[attend(x, x, x, pos, None, slope)] * 3, pos, None, slope)}[case]
    _both_ways(function, [x, pos, slope], gen, 1e-5)        # fp32: some hundred roundings of 2^-24


def test_expression_of_the_feed_forward_block():
    from equitorch_amd.nn.functional.feed_forward import _expression
    gen = torch.Generator().manual_seed(3)
    leaves = [_rand(gen, *s, dtype=F32, std=0.5).requires_grad_(True) for s in ((7, 6), (6, 9), (9, 6))]
    block = lambda x, w, d: _as_operator(_expression(0), (x, w, w, d))
    _both_ways(lambda x, w, d: block(block(x, w, d), w, d), leaves, gen, 1e-5)


# ---- the operators ----------------------------------------------------------------------------------------------------
@pytest.fixture(params=[True, False], ids=["extension", "ctypes"])
def extension(request, monkeypatch):
    from equitorch_amd import _shim
    assert _shim.module() is not None
    if not request.param:
        monkeypatch.setattr(_shim, "_module", None)


@gpu
@pytest.mark.parametrize("case", ["one tensor", "keys and values", "layers"])
def test_attention(device, extension, case):
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    gen = torch.Generator().manual_seed(4)
    plan = AttentionPlan(torch.tensor([0, 20, 20, 75], device=device))
    x, pos, slope = (t.to(device).requires_grad_(True) for t in (_rand(gen, 75, 4, 16, dtype=F32), _rand(gen, 75, 3, dtype=F32),
                                                                  torch.rand(4, generator=gen)))
    attend = lambda q, k, v, pos, slope, pos_k=None: segment_attention(q, k, v, plan, pos=pos, slope=slope, pos_k=pos_k, cap=5.0)
    function = {"one tensor": lambda x, pos, slope: attend(x, x, x, pos, slope),
                "keys and values": lambda x, pos, slope: attend(x, x * 2.0, x * 2.0, pos, slope, pos),
                "layers": lambda x, pos, slope: attend(*[attend(x, x, x, pos, slope)] * 3, pos, slope)}[case]
    _both_ways(function, [x, pos, slope], gen, 1e-4)        # fp32 either way, sums over up to 55 keys in other orders


@gpu
def test_feed_forward_blocks_that_share_weights(device, extension):
    from equitorch_amd.nn.functional import gated_feed_forward
    gen = torch.Generator().manual_seed(5)
    leaves = [_rand(gen, *s, dtype=F32, std=0.2).to(device).requires_grad_(True) for s in ((50, 32), (32, 40), (40, 32))]
    block = lambda x, w, d: gated_feed_forward(x, w, w, d)
    _both_ways(lambda x, w, d: block(block(x, w, d), w, d), leaves, gen, 1e-4)


@gpu
@pytest.mark.parametrize("mode", ["harmonics", "vectors", "radial", "table", "shared weight"])
def test_edge_products_that_share_harmonics_and_weights(device, extension, mode):
    from equitorch_amd.nn import SO3Linear
    from equitorch_amd.nn.functional import (EdgePlan, edge_tensor_product_uu, edge_tensor_product_uu_radial,
                                             edge_tensor_product_uu_vectors)
    irreps = "0e+1o" if mode == "table" else "0e+1o+2e"
    i2, ch, n, e, r = "0e+1o+2e", 32 if mode == "table" else 64, 30, 300, 8
    mod = SO3Linear(irreps, i2, irreps, ch, ch, internal_weights=False, feature_mode="uu").to(device)
    gen = torch.Generator().manual_seed(6)
    plan = EdgePlan(*(torch.randint(0, n, (e,), generator=gen).to(device) for _ in range(2)), n)
    shapes = [(n, 4 if mode == "table" else 9, ch), (e, 3) if mode == "vectors" else (e, 9)]
    shapes += [(e, r), (r, mod.num_paths, ch)] if mode == "radial" else [(mod.num_paths, ch) if mode == "shared weight" else (e, mod.num_paths, ch)]
    leaves = [_rand(gen, *s, dtype=F32, std=0.3 if i else 1.0).to(device).requires_grad_(True) for i, s in enumerate(shapes)]

    def layer(x, y, *w):
        if mode == "radial":
            return edge_tensor_product_uu_radial(x, y, *w, plan, mod.tp_info_forward)
        if mode == "vectors":
            return edge_tensor_product_uu_vectors(x, y, *w, plan, mod.tp_info_forward)
        return edge_tensor_product_uu(x, y, *w, plan, mod.tp_info_forward)
    _both_ways(lambda x, *rest: layer(layer(x, *rest) * 0.3, *rest), leaves, gen, 1e-4)


@gpu
def test_norm_rotation_and_radial_functions(device):
    from equitorch_amd.nn import LayerRMSNorm, SparseWignerRotation
    from equitorch_amd.nn.functional import _radial, layer_rms_norm, sincos
    gen = torch.Generator().manual_seed(7)
    norm = LayerRMSNorm("0e+1o+2e", 32).to(device)
    x, angles = _rand(gen, 40, 9, 32).to(device), [_rand(gen, 40).to(device) for _ in range(3)]
    weight = (torch.rand(3, 32, generator=gen, dtype=F64) + 0.5).to(device).requires_grad_(True)
    twice = lambda x, w: layer_rms_norm(layer_rms_norm(x, norm.irreps_info, w) + x, norm.irreps_info, w)
    _both_ways(twice, [x.requires_grad_(True), weight], gen, 1e-10)
    rotation = SparseWignerRotation("0e+1o+2e").to(device)
    leaves = [x] + [sincos(a, 2).detach().requires_grad_(True) for a in angles]
    _both_ways(lambda x, a, b, c: rotation(torch.tanh(rotation(x, a, b, c)), a, b, c), leaves, gen, 1e-10)
    r = (torch.rand(50, generator=gen, dtype=F64) * 2 + 0.5).to(device).requires_grad_(True)
    expression = lambda r, f: (2 / 3.0) * torch.sin(f * r[..., None] / 3.0) / r[..., None]
    _both_ways(lambda r: _radial.bessel(r, r[:4] * 2.0, 3.0, expression), [r], gen, 1e-10)


@gpu
@pytest.mark.parametrize("mode", ["u1v", "u1v per sample", "vu1", "uvw", "uuu", "u1u"])
def test_products_that_share_operands(device, mode):
    import equitorch_amd.nn.functional as F
    from equitorch_amd.irreps import Irreps
    from equitorch_amd.utils import tp_infos
    irr = Irreps("0e+1o")
    infos = [t.to(device) for t in tp_infos(irr, irr, irr)[:3]]
    p, n, c, gen = 4, 40, 16, torch.Generator().manual_seed(8)
    rd = lambda *s: _rand(gen, *s, std=0.5).to(device).requires_grad_(True)
    x, y = rd(n, 4, c), rd(n, 4)
    if mode.startswith("u1v"):
        w = rd(n, p, c, c) if "sample" in mode else rd(p, c, c)
        layer = lambda x, y, w: F.tensor_product_u1v(x, y, w, *infos)
        _both_ways(lambda x, y, w: layer(layer(x, y, w), y, w), [x, y, w], gen, 1e-10)
    elif mode == "vu1":
        w = rd(p, c, c)
        _both_ways(lambda x, w: F.tensor_product_vu1(x, x * 2.0, w, *infos), [x, w], gen, 1e-10)
    elif mode == "uvw":
        w = rd(p, c, c, c)
        layer = lambda x, w: F.tensor_product_uvw(x, x, w, *infos)
        _both_ways(lambda x, w: layer(layer(x, w), w), [x, w], gen, 1e-10)
    elif mode == "uuu":
        w = rd(p, c)
        layer = lambda x, w: F.tensor_product_uuu(x, x, w, *infos)
        _both_ways(lambda x, w: layer(layer(x, w), w), [x, w], gen, 1e-10)
    else:
        w = rd(n, p, c)
        layer = lambda x, y, w: F.tensor_product_u1u(x, y, w, *infos)
        _both_ways(lambda x, y, w: layer(layer(x, y, w), y, w), [x, y, w], gen, 1e-10)


@gpu
def test_example_forces_in_the_loss(device):
    """Forces under ``create_graph`` and what a loss on them and on the energies sends back to every parameter, against
    the same model from its definition in 64 bits.  Two layers share the positions."""
    from test_gpu_node_modules import _attend, _example, _feed
    ex = _example()
    torch.manual_seed(9)
    kind, pos, ptr = ex.make_structures(5, torch.Generator().manual_seed(9), device)
    model = ex.StructureEnergy().to(device)
    energy, forces = model.energy_and_forces(kind, pos, ptr, create_graph=True)
    gen = torch.Generator().manual_seed(10)
    ct, cf = _rand(gen, *energy.shape), _rand(gen, *forces.shape)
    names, weights = zip(*model.named_parameters())
    got = torch.autograd.grad((energy * ct.to(energy)).sum() + (forces * cf.to(forces)).sum(), weights, allow_unused=True)

    wide = ex.StructureEnergy()
    wide.load_state_dict(model.state_dict())
    wide = wide.double()
    norm = lambda m, x: x * (x.square().mean(-1, keepdim=True) + m.eps).rsqrt() * m.weight
    p, at = pos.double().cpu().requires_grad_(True), ptr.tolist()
    x = wide.embedding.weight[kind.cpu()]
    for layer in wide.layers:
        x = x + _attend(layer.attention, norm(layer.norm1, x), at, p)
        x = x + _feed(layer.feed_forward, norm(layer.norm2, x))
    q = wide.query.expand(len(at) - 1, -1)
    out = _attend(wide.readout, q, list(range(len(at))), None, norm(wide.norm, x), at)
    e = (out @ wide.head.weight.T + wide.head.bias)[:, 0] * torch.diff(ptr).cpu()
    (grad,) = torch.autograd.grad(e.sum(), p, create_graph=True)
    want = torch.autograd.grad((e * ct).sum() - (grad * cf).sum(), list(wide.parameters()), allow_unused=True)
    # fp32 through two layers and two orders: as for energies and forces without a loss on them, 2e-3 of the largest element
    for name, a, b in zip(("energy", "forces", *names), (energy, forces, *got), (e, -grad, *want)):
        if a is None or b is None:
            assert a is b, name
            continue
        worst = float((a.detach().cpu().double() - b.detach()).abs().max())
        assert worst <= 2e-3 * max(1.0, float(b.abs().max())), f"{name}: {worst:.3e}"


LENGTHS_OF_NOTHING = [([], []), ([0, 0], [0, 0]), ([0, 0], [3, 40]), ([2, 40], [0, 0])]


@pytest.mark.parametrize("len_q,len_k", LENGTHS_OF_NOTHING)
def test_expression_of_the_attention_of_nothing(len_q, len_k):
    """No queries, or no keys: gradients of zeros, not none."""
    from equitorch_amd.nn.functional import AttentionPlan
    from equitorch_amd.nn.functional.attention import _of_buckets
    ptr = lambda n: torch.tensor([0] + n).cumsum(0)
    t = [torch.ones(sum(n), h, 4, requires_grad=True) for n, h in ((len_q, 2), (len_k, 1), (len_k, 1))]
    t += [torch.ones(sum(n), 3, requires_grad=True) for n in (len_q, len_k)] + [torch.ones(2, requires_grad=True)]
    got = higher_order(_of_buckets(AttentionPlan(ptr(len_q), ptr(len_k))._buckets, 1.0, 0.0), t, [True] * 6, torch.ones_like(t[0]))
    for a, b in zip(got, t):
        assert torch.equal(a, torch.zeros_like(b))


@gpu
@pytest.mark.parametrize("len_q,len_k", LENGTHS_OF_NOTHING)
@pytest.mark.parametrize("create_graph", [False, True])
def test_attention_of_nothing(device, extension, len_q, len_k, create_graph):
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    ptr = lambda n: torch.tensor([0] + n, device=device).cumsum(0)
    t = [torch.ones(sum(n), h, 4, device=device, requires_grad=True) for n, h in ((len_q, 2), (len_k, 1), (len_k, 1))]
    pos, pos_k = (torch.ones(sum(n), 3, device=device, requires_grad=True) for n in (len_q, len_k))
    t += [pos, pos_k, torch.ones(2, device=device, requires_grad=True)]
    out = segment_attention(*t[:3], AttentionPlan(ptr(len_q), ptr(len_k)), pos=pos, slope=t[5], pos_k=pos_k)
    assert torch.equal(out, torch.zeros_like(t[0]))
    for a, b in zip(torch.autograd.grad(out.sum(), t, create_graph=create_graph), t):
        assert torch.equal(a, torch.zeros_like(b))


def test_expression_of_the_attention_with_nodes_beyond_any_distance():
    """A squared distance beyond fp32: that node takes no part, in the gradients either, of first and second order."""
    from equitorch_amd.nn.functional import AttentionPlan
    from equitorch_amd.nn.functional.attention import _of_buckets
    gen = torch.Generator().manual_seed(11)
    near = slice(0, 9)
    data = [_rand(gen, 10, 2, 4, dtype=F32) for _ in range(3)] + [_rand(gen, 10, 3, dtype=F32), torch.rand(2, generator=gen) + 0.1]
    data[3][9] = torch.tensor([1e20, 0.0, -2e20])
    ct, cf = _rand(gen, 10, 2, 4, dtype=F32), _rand(gen, 10, 3, dtype=F32)
    seen = []
    for n in (10, 9):
        t = [a[:n].clone().requires_grad_(True) for a in data[:4]] + [data[4].clone().requires_grad_(True)]
        q, k, v, pos, slope = t
        out = _as_operator(_of_buckets(AttentionPlan(torch.tensor([0, n]))._buckets, 0.5, 0.0), (q, k, v, pos, None, slope))
        first = torch.autograd.grad(out[near], t, ct[near], create_graph=True)
        second = torch.autograd.grad((first[3][near] * cf[near]).sum(), t)
        seen.append([out, *first, *second])
    for a, b in zip(*seen):                                # the nine others: sums of ten terms in another order
        assert torch.isfinite(a).all()
        a = a[near] if a.shape[0] == 10 else a
        assert float((a - b).detach().abs().max()) <= 1e-5 * max(1.0, float(b.detach().abs().max()))


@gpu
@pytest.mark.parametrize("fused", [False, True])
def test_layer_whose_weights_come_from_the_edge_vectors(device, extension, fused):
    """A message-passing layer as models have it: radial functions of the edge vectors make the weights of a product that takes
    the vectors too, twice over."""
    from equitorch_amd import nn as enn
    from equitorch_amd.nn.functional import EdgePlan, edge_tensor_product_uu_radial, edge_tensor_product_uu_vectors
    irr, n, e, c = "0e+1o+2e", 30, 300, 64
    torch.manual_seed(12)
    gen = torch.Generator().manual_seed(12)
    tp = enn.SO3Linear(irr, irr, irr, c, c, internal_weights=False, feature_mode="uu").to(device)
    basis, cutoff = enn.BesselBasis(3.0, 8).to(device), enn.PolynomialCutoff(3.0)
    hidden = torch.nn.Sequential(torch.nn.Linear(8, 16), torch.nn.SiLU()).to(device)
    mix, gate_lin, gate, norm = (m.to(device) for m in (enn.IrrepsLinear(irr, irr, c, c), enn.IrrepsLinear(irr, "0e+0e+0e", c, c),
                                                        enn.Gate(irr, activation=torch.nn.Sigmoid()), enn.LayerRMSNorm(irr, c)))
    plan = EdgePlan(*(torch.randint(0, n, (e,), generator=gen).to(device) for _ in range(2)), n)
    x, vec, last = (_rand(gen, *s, dtype=F32, std=0.5).to(device).requires_grad_(True) for s in ((n, 9, c), (e, 3), (16, tp.num_paths, c)))

    def layer(x, vec, last):
        r = vec.norm(dim=-1)
        feat = hidden(basis(r) * cutoff(r)[:, None])
        if fused:
            msg = edge_tensor_product_uu_radial(x, vec, feat, last, plan, tp.tp_info_forward, edge_vectors=True)
        else:
            msg = edge_tensor_product_uu_vectors(x, vec, (feat @ last.reshape(16, -1)).view(e, -1, c), plan, tp.tp_info_forward)
        h = mix(msg)
        return norm(gate(h, gate_lin(h)))
    # fp32 through two layers; gradients of a length near zero are large
    _both_ways(lambda x, vec, last: layer(layer(x, vec, last) + x, vec, last), [x, vec, last], gen, 1e-3)
