"""Embedding of node kinds, attention among the nodes of a structure and the gated feed-forward block against plain
implementations in 64 bits on the CPU.

Tolerances are bounds on rounding, element by element: the result's own rounding, plus a number of roundings of what the
kernels hold in fewer bits times the sum of the magnitudes that enter the element (the same formula with absolute values)."""
import pytest
import torch

from equitorch_amd._lib import CgtpError
from helpers import stable_seed

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
EPS = {F64: 2.0 ** -53, F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}      # half a unit in the last place
TINY = {F64: 0.0, F32: 1e-37, BF16: 1e-37, F16: 2.0 ** -24}                      # below: subnormal


def _rand(gen, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=gen, dtype=F64) * std).to(dtype)


def _within(got, want, bound, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} vs {tuple(want.shape)}"
    excess = ((got - want).abs() - bound).max() if want.numel() else torch.tensor(-1.0)
    assert float(excess) <= 0 and torch.isfinite(got).all(), f"{what}: {float(excess):.3e} over the bound"


# ---- embedding ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("rows,kinds,channels", [(1, 1, 1), (30, 100, 64), (257, 3, 7), (5000, 255, 33), (4099, 256, 128),
                                                 (20011, 1000, 24), (9000, 70001, 16), (130001, 5, 8), (700, 90, 1200)])
def test_embedding(device, dtype, rows, kinds, channels):
    from equitorch_amd.nn.functional import embedding
    gen = torch.Generator().manual_seed(stable_seed(rows, kinds, channels))
    # a few kinds hold most rows; a kind below zero and one beyond the table give zeros
    kind = (torch.rand(rows, generator=gen, dtype=F64) ** 3 * kinds).long()
    if rows > 20:
        kind[3], kind[rows // 2] = -1, kinds
    table, ct = _rand(gen, kinds, channels, dtype=dtype), _rand(gen, rows, channels, dtype=dtype)
    scale = channels ** 0.5
    t = table.to(device).requires_grad_(True)
    out = embedding(kind.to(device), t, scale)
    (grad,) = torch.autograd.grad(out, t, ct.to(device))
    ok = ((kind >= 0) & (kind < kinds)).double()[:, None]
    at = kind.clamp(0, kinds - 1)
    want = table.double()[at] * scale * ok
    unit = EPS[F64] if dtype == F64 else EPS[F32]
    _within(out, want, (EPS[dtype] + 2 * unit) * want.abs() + TINY[dtype], "out")
    sums, size = torch.zeros(kinds, channels, dtype=F64), torch.zeros(kinds, channels, dtype=F64)
    sums.index_add_(0, at, ct.double() * scale * ok)
    size.index_add_(0, at, (ct.double() * scale * ok).abs())
    # the chunks' sums and their sum: no element is added in a chain longer than its kind's rows
    count = torch.bincount(at, minlength=kinds).double()[:, None]
    _within(grad, sums, EPS[dtype] * sums.abs() + (count + 4) * unit * size + TINY[dtype], "grad")
    (again,) = torch.autograd.grad(embedding(kind.to(device), t, scale), t, ct.to(device))
    assert torch.equal(again, grad)


def test_embedding_shapes_and_second_order(device):
    from equitorch_amd.nn.functional import embedding
    gen = torch.Generator().manual_seed(5)
    kind = torch.randint(0, 9, (4, 5), generator=gen)
    table = _rand(gen, 9, 6).to(device).requires_grad_(True)
    assert embedding(kind.to(device), table).shape == (4, 5, 6)
    assert embedding(torch.zeros(0, dtype=torch.int64, device=device), table).shape == (0, 6)
    (empty,) = torch.autograd.grad(embedding(torch.zeros(0, dtype=torch.int64, device=device), table).sum(), table)
    assert torch.equal(empty, torch.zeros_like(empty))
    # an unaligned table: rows from an offset that is no multiple of 16 bytes
    loose = torch.empty(9 * 6 + 1, device=device)[1:].view(9, 6).copy_(table.detach()).requires_grad_(True)
    assert torch.equal(embedding(kind.to(device), loose), embedding(kind.to(device), table))
    ct = _rand(gen, 4, 5, 6).to(device).requires_grad_(True)
    (g,) = torch.autograd.grad(embedding(kind.to(device), table, 2.0), table, ct, create_graph=True)
    v = _rand(gen, 9, 6).to(device)
    (gg,) = torch.autograd.grad((g * v).sum(), ct)
    assert torch.equal(gg, 2.0 * v[kind.to(device)])


def test_embedding_refuses(device):
    from equitorch_amd.nn.functional import embedding
    kind, table = torch.zeros(3, dtype=torch.int64, device=device), torch.zeros(4, 5, device=device)
    for bad in ((kind.int(), table), (kind, table[0]), (kind, table.long()), (kind, table[:0]), (kind.cpu(), table),
                (kind, table.cpu())):
        with pytest.raises(CgtpError):
            embedding(*bad)


# ---- attention ---------------------------------------------------------------------------------------------------
def _reference(q, k, v, len_q, len_k, pos, pos_k, slope, scale, cap, ct):
    """``{name: (value, bound on rounding in units)}``: the magnitudes are sums of absolute values, once for what is rounded
    to the operands' type and once for what errs in fp32 (the scores)."""
    q, k, v, ct = (t.double() for t in (q, k, v, ct))
    group = q.shape[1] // k.shape[1]
    z = torch.zeros_like
    names = ("out", "q", "k", "v")
    val = {"out": z(q), "q": z(q), "k": z(k), "v": z(v)}
    mag = {n: z(t) for n, t in val.items()}
    if slope is not None:
        pos, pos_k, slope = pos.double(), pos_k.double(), slope.double()
        for n, t in (("pos", pos), ("pos_k", pos_k), ("slope", slope)):
            val[n], mag[n] = z(t), z(t)
    top = 0.0
    a = b = 0
    for lq, lk in zip(len_q, len_k):
        rq, rk = slice(a, a + lq), slice(b, b + lk)
        a, b = a + lq, b + lk
        if not lq or not lk:
            continue
        for h in range(q.shape[1]):
            hk = h // group
            x = q[rq, h] @ k[rk, hk].T * scale
            th = torch.tanh(x / cap) if cap else z(x)
            s = cap * th if cap else x
            if slope is not None:
                delta = pos[rq, None] - pos_k[None, rk]
                dist = delta.norm(dim=-1)
                unit = torch.where(dist[..., None] > 0, delta / dist[..., None].clamp(min=1e-300), z(delta))
                s = s - slope[h] * dist
            top = max(top, float(s.abs().max()), float((q[rq, h].abs() @ k[rk, hk].abs().T * scale).max()))
            p = torch.softmax(s, 1)
            o = p @ v[rk, hk]
            val["out"][rq, h], mag["out"][rq, h] = o, p @ v[rk, hk].abs()
            g = ct[rq, h]
            dp = g @ v[rk, hk].T
            ds = p * (dp - (p * dp).sum(1, keepdim=True))
            size = p * (g.abs() @ v[rk, hk].abs().T + (g.abs() * mag["out"][rq, h]).sum(1, keepdim=True))
            val["v"][rk, hk] += p.T @ g
            mag["v"][rk, hk] += p.T @ g.abs()
            if slope is not None:
                val["slope"][h] -= (ds * dist).sum()
                mag["slope"][h] += (size * dist).sum()
                pull, most = -slope[h] * ds[..., None] * unit, slope[h].abs() * size[..., None] * unit.abs()
                val["pos"][rq] += pull.sum(1)
                mag["pos"][rq] += most.sum(1)
                val["pos_k"][rk] -= pull.sum(0)
                mag["pos_k"][rk] += most.sum(0)
            ds = ds * (1 - th * th)
            val["q"][rq, h], mag["q"][rq, h] = scale * ds @ k[rk, hk], scale * size @ k[rk, hk].abs()
            val["k"][rk, hk] += scale * ds.T @ q[rq, h]
            mag["k"][rk, hk] += scale * size.T @ q[rq, h].abs()
    return val, mag, top


LENGTHS = {
    "one": ([1], [1]),
    "short": ([3, 0, 1, 17, 31, 32, 33, 2], None),
    "odd": ([65, 130, 7, 64, 1], None),
    "long": ([700], None),
    "readout": ([1, 1, 1, 1, 0], [5, 0, 63, 300, 4]),
    "one_long": ([1], [5003]),
    "few_keys": ([1500, 2], [3, 1]),
    "mixed": ([129, 0, 40], [0, 9, 260]),
}


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,biased,cap", [
    ("one", 1, 1, 1, True, 0.0), ("short", 8, 8, 16, True, 0.0), ("short", 6, 2, 13, True, 5.0), ("odd", 4, 4, 32, True, 4.0),
    ("odd", 4, 1, 64, False, 0.0), ("long", 2, 1, 72, True, 3.0), ("long", 2, 2, 128, False, 0.0), ("readout", 8, 8, 32, True, 0.0),
    ("readout", 8, 2, 64, False, 2.0), ("one_long", 8, 2, 64, True, 30.0), ("one_long", 2, 2, 100, False, 0.0),
    ("few_keys", 4, 2, 24, True, 0.0), ("mixed", 3, 3, 96, True, 6.0), ("mixed", 4, 4, 8, False, 0.0)])
def test_attention(device, dtype, lengths, heads, kv_heads, dim, biased, cap):
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    len_q, len_k = LENGTHS[lengths]
    own = len_k is None
    len_k = len_q if own else len_k
    nq, nk = sum(len_q), sum(len_k)
    gen = torch.Generator().manual_seed(stable_seed(lengths, heads, kv_heads, dim))
    # slices of wider tensors: rows, heads and the start of a row lie anywhere
    q = _rand(gen, nq, heads + 1, dim + 3, dtype=dtype)
    kv = _rand(gen, nk, 2 * kv_heads, dim + 1, dtype=dtype)
    ct = _rand(gen, nq, heads, dim, dtype=dtype)
    pos = _rand(gen, nq, 3, std=2.0) if biased else None
    pos_k = (pos if own else _rand(gen, nk, 3, std=2.0)) if biased else None
    slope = torch.rand(heads, generator=gen) if biased else None
    cut = lambda q, kv: (q[:, 1:, 2:dim + 2], kv[:, :kv_heads, 1:], kv[:, kv_heads:, 1:])
    scale = dim ** -0.5
    val, mag, top = _reference(*cut(q, kv), len_q, len_k, pos, pos_k, slope, scale, cap, ct)

    ptr = lambda n: torch.tensor([0] + n, device=device).cumsum(0)
    plan = AttentionPlan(ptr(len_q)) if own else AttentionPlan(ptr(len_q), ptr(len_k))
    leaves = [t.detach().requires_grad_(True) for t in cut(q.to(device), kv.to(device))]
    more = [None if t is None else t.to(device).requires_grad_(True) for t in (pos, None if own else pos_k, slope)]
    run = lambda: segment_attention(*leaves, plan, pos=more[0], pos_k=more[1], slope=more[2], cap=cap or None)
    out = run()
    wrt = leaves + [t for t in more if t is not None]
    grads = torch.autograd.grad(out, wrt, ct.to(device))
    names = ["q", "k", "v"] + [n for n, t in zip(("pos", "pos_k", "slope"), more) if t is not None]
    if biased and own:
        val["pos"], mag["pos"] = val["pos"] + val["pos_k"], mag["pos"] + mag["pos_k"]
    # 16-bit: the probability, the score's gradient, the output inside delta and one more rounding of each term; fp32: the sums
    # over dim and the keys, and the score's error, which moves every probability
    unit = 4 * EPS[dtype] + EPS[F32] * (32 + dim + 16 * top) if dtype != F32 else EPS[F32] * (32 + dim + 16 * top)
    for name, got in zip(["out"] + names, [out, *grads]):
        own_type = EPS[F32] if name in ("pos", "pos_k", "slope") else EPS[dtype]
        _within(got, val[name], own_type * val[name].abs() + unit * mag[name] + 64 * TINY[dtype], name)
    again = torch.autograd.grad(run(), wrt, ct.to(device))
    assert all(torch.equal(a, b) for a, b in zip(again, grads))
    with torch.no_grad():
        assert torch.equal(run(), out)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_structures_do_not_touch(device, dtype, bad):
    """What one structure holds does not reach another, whatever it is."""
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    gen = torch.Generator().manual_seed(3)
    lengths = [9, 20, 70, 5]
    n = sum(lengths)
    plan = AttentionPlan(torch.tensor([0] + lengths, device=device).cumsum(0))
    data = [_rand(gen, n, 2, 32, dtype=dtype).to(device) for _ in range(4)]
    pos, slope = _rand(gen, n, 3).to(device), torch.rand(2, generator=gen).to(device)

    def run(tensors, pos):
        q, k, v = (t.clone().requires_grad_(True) for t in tensors[:3])
        p = pos.clone().requires_grad_(True)
        out = segment_attention(q, k, v, plan, pos=p, slope=slope)
        return (out, *torch.autograd.grad(out, (q, k, v, p), tensors[3]))
    clean = run(data, pos)
    rows = slice(9, 29)                                    # the second structure
    spoiled = [t.clone() for t in data]
    for t in spoiled:
        t[rows] = bad
    p = pos.clone()
    p[rows] = bad
    keep = torch.ones(n, dtype=torch.bool, device=device)
    keep[rows] = False
    for a, b in zip(clean, run(spoiled, p)):
        assert torch.equal(a[keep], b[keep])


def test_attention_scores_out_of_range(device):
    """Scores of -inf mask a key; a row of nothing else is zeros, and so are its gradients."""
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    q = torch.ones(4, 1, 8, device=device).requires_grad_(True)
    k = torch.ones(4, 1, 8, device=device)
    k[2:] = -torch.inf
    v = torch.arange(32.0, device=device).view(4, 1, 8)
    plan = AttentionPlan(torch.tensor([0, 3, 4], device=device))
    out = segment_attention(q, k, v, plan)
    assert torch.equal(out[:3, 0], v[:2, 0].mean(0).expand(3, 8)) and torch.equal(out[3], torch.zeros_like(out[3]))
    finite = torch.full((4, 1, 8), -3.0e38, device=device)
    far = segment_attention(q.detach() * 1e3, finite, v, plan)      # every score the lowest of the type, or -inf
    assert torch.isfinite(far).all()


def test_attention_differences(device):
    """Gradients of a scalar against differences of the forward itself, and second order against differences of the first."""
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    gen = torch.Generator().manual_seed(11)
    lengths = [5, 0, 12]
    n = sum(lengths)
    plan = AttentionPlan.from_batch(torch.repeat_interleave(torch.arange(3), torch.tensor(lengths)).to(device), 3)
    data = [_rand(gen, n, 4, 16), _rand(gen, n, 2, 16), _rand(gen, n, 2, 16), _rand(gen, n, 3), torch.rand(4, generator=gen)]
    step = [_rand(gen, *t.shape) for t in data]
    ct = _rand(gen, n, 4, 16).to(device)

    def value(eps, create_graph=False):
        x = [(t + eps * d).to(device).requires_grad_(True) for t, d in zip(data, step)]
        out = segment_attention(*x[:3], plan, pos=x[3], slope=x[4], cap=4.0)
        return x, (out * ct).sum().double() if not create_graph else (out * ct).sum()

    x, y = value(0.0, True)
    grads = torch.autograd.grad(y, x, create_graph=True)
    along = sum((g.double() * d.to(device).double()).sum() for g, d in zip(grads, step))
    eps = 2.0 ** -7          # error eps^2 of the difference and 2^-24 * sqrt(sum) / eps of the values
    diff = (value(eps)[1] - value(-eps)[1]) / (2 * eps)
    assert abs(float(diff - along)) <= 5e-3 * (1 + abs(float(along)))
    # second order: the gradient's change along the step
    second = torch.autograd.grad(along, x)

    def gradient(eps):
        x, y = value(eps, True)
        return torch.autograd.grad(y, x)
    up, down = gradient(eps), gradient(-eps)
    for s, a, b in zip(second, up, down):
        want = (a.double() - b.double()) / (2 * eps)
        assert float((s.double() - want).abs().max()) <= 2e-2 * (1 + float(want.abs().max()))


def test_attention_refuses(device):
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    ptr = torch.tensor([0, 2, 6], device=device)
    plan = AttentionPlan(ptr)
    q, k, v = (torch.zeros(6, 2, 8, device=device) for _ in range(3))
    pos, slope = torch.zeros(6, 3, device=device), torch.zeros(2, device=device)
    segment_attention(q, k, v, plan, pos=pos, slope=slope, cap=1.0)
    wrong = torch.zeros(6, 3, 8, device=device)
    wide = torch.zeros(6, 2, 130, device=device)
    for args, kw in (((q[:5], k, v, plan), {}), ((q, k[:5], v[:5], plan), {}), ((q, wrong, wrong, plan), {}), ((q, k, v[:, :1], plan), {}),
                     ((wide, wide, wide, plan), {}), ((q.double(), k.double(), v.double(), plan), {}), ((q, k.bfloat16(), v, plan), {}),
                     ((q.cpu(), k, v, plan), {}), ((q, k, v, plan), {"pos": pos}), ((q, k, v, plan), {"slope": slope}),
                     ((q, k, v, plan), {"slope": slope[:1], "pos": pos}), ((q, k, v, plan), {"slope": slope, "pos": pos[:, :2]}),
                     ((q, k, v, plan), {"slope": slope.double(), "pos": pos}), ((q, k, v, plan), {"cap": -1.0}),
                     ((q, k, v, plan), {"cap": float("inf")}), ((q, k, v, plan), {"cap": float("nan")}),
                     ((q, k, v, AttentionPlan(ptr, ptr)), {"slope": slope, "pos": pos})):
        with pytest.raises(CgtpError):
            segment_attention(*args, **kw)


def test_attention_under_a_stream_and_a_graph(device):
    from equitorch_amd.nn.functional import AttentionPlan, embedding, gated_feed_forward, segment_attention
    gen = torch.Generator().manual_seed(7)
    n = 90
    kind, table = torch.randint(0, 9, (n,), generator=gen).to(device), _rand(gen, 9, 64).to(device)
    plan = AttentionPlan(torch.tensor([0, 50, n], device=device))
    pos, slope = _rand(gen, n, 3).to(device), torch.rand(2, generator=gen).to(device)
    w = [_rand(gen, *s, std=0.1).to(device) for s in ((64, 96), (64, 96), (96, 64))]

    def step(pos):
        t = [x.detach().requires_grad_(True) for x in (table, pos, *w)]
        x = embedding(kind, t[0]).view(n, 2, 32)
        y = gated_feed_forward(segment_attention(x, x, x, plan, pos=t[1], slope=slope).reshape(n, 64), *t[2:])
        return (y, *torch.autograd.grad((y * y).sum(), t))
    want = [step(pos), step(2 * pos)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(pos)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graph, given = torch.cuda.CUDAGraph(), pos.clone()
    with torch.cuda.graph(graph):
        kept = step(given)
    for i in (0, 1, 0):
        given.copy_((1 + i) * pos)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want[i]))
        step(pos)                              # eager work between the replays


# ---- gated feed-forward --------------------------------------------------------------------------------------------
def _act64(name, u):
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(u / 2 ** 0.5))
        return u * cdf, cdf + u * torch.exp(-u * u / 2) / (2 * torch.pi) ** 0.5
    s = torch.sigmoid(u)
    return (u * s, s + u * s * (1 - s)) if name == "silu" else (s, s * (1 - s))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,c,h,co,activation", [(1, 256, 1024, 256, "silu"), (1, 1, 1, 1, "silu"), (7, 16, 33, 5, "gelu"),
                                                    (16, 128, 512, 128, "silu"), (33, 70, 129, 65, "sigmoid"),
                                                    (129, 129, 64, 130, "silu"), (1000, 64, 256, 64, "gelu"),
                                                    (5003, 40, 72, 24, "silu"), (640, 256, 130, 256, "silu")])
def test_gated_feed_forward(device, dtype, rows, c, h, co, activation):
    from equitorch_amd.nn.functional import gated_feed_forward
    gen = torch.Generator().manual_seed(stable_seed(rows, c, h, co))
    x, ct = _rand(gen, rows, c, dtype=dtype), _rand(gen, rows, co, dtype=dtype)
    ws = [_rand(gen, c, h, dtype=dtype, std=c ** -0.5), _rand(gen, c, h, dtype=dtype, std=c ** -0.5),
          _rand(gen, h, co, dtype=dtype, std=h ** -0.5)]
    leaves = [t.to(device).requires_grad_(True) for t in (x, *ws)]
    out = gated_feed_forward(*leaves, activation)
    grads = torch.autograd.grad(out, leaves, ct.to(device))
    xd, gd, (wg, wu, wd) = x.double(), ct.double(), (t.double() for t in ws)
    u, r = xd @ wg, xd @ wu
    act, slope = _act64(activation, u)
    mid = act * r
    dm = gd @ wd.T
    dg, du = dm * r * slope, dm * act
    want = (mid @ wd, dg @ wg.T + du @ wu.T, xd.T @ dg, xd.T @ du, mid.T @ gd)
    # magnitudes of what each factor errs by in units: the projections over their sums' sizes, the rest over its own
    su, sr = xd.abs() @ wg.abs(), xd.abs() @ wu.abs()
    sm = act.abs() * sr + 1.2 * su * r.abs()
    sd = gd.abs() @ wd.abs().T
    sg, sdu = sd * (r.abs() + sr) * 1.2 + dm.abs() * r.abs() * su, sd * act.abs() + dm.abs() * 1.2 * su
    size = (sm @ wd.abs(), sg @ wg.abs().T + sdu @ wu.abs().T, xd.abs().T @ sg, xd.abs().T @ sdu, sm.T @ gd.abs())
    # 16-bit: the projections, the product and its gradients are rounded once each; fp32: sums over the longest axis
    unit = 4 * EPS[dtype] if dtype != F32 else EPS[F32] * (16 + max(c, h, co, rows) ** 0.5)
    for name, got, w, s in zip(("out", "x", "w_gate", "w_up", "w_down"), (out, *grads), want, size):
        _within(got, w, EPS[dtype] * w.abs() + unit * s + 64 * TINY[dtype], name)
    with torch.no_grad():
        assert torch.equal(gated_feed_forward(*leaves, activation), out)
    again = torch.autograd.grad(gated_feed_forward(*leaves, activation), leaves, ct.to(device))
    assert all(torch.equal(a, b) for a, b in zip(again, grads))


def test_gated_feed_forward_layouts_and_higher_order(device):
    from equitorch_amd.nn.functional import gated_feed_forward
    gen = torch.Generator().manual_seed(9)
    x, ws = _rand(gen, 3, 4, 10).to(device), [_rand(gen, *s, std=0.3).to(device) for s in ((10, 12), (10, 12), (12, 6))]
    out = gated_feed_forward(x, *ws)
    assert out.shape == (3, 4, 6)
    # transposed weights and a strided x give the same
    same = gated_feed_forward(x.transpose(0, 1).contiguous().transpose(0, 1), *[w.T.contiguous().T for w in ws])
    assert torch.equal(out, same)
    assert gated_feed_forward(x[:0], *ws).shape == (0, 4, 6)
    leaves = [t.detach().requires_grad_(True) for t in (x[:0], *ws)]
    for g in torch.autograd.grad(gated_feed_forward(*leaves).sum(), leaves):
        assert torch.equal(g, torch.zeros_like(g))
    # only some gradients wanted
    w_only = [x, ws[0].detach().requires_grad_(True), ws[1], ws[2].detach().requires_grad_(True)]
    part = torch.autograd.grad(gated_feed_forward(*w_only).sum(), [w_only[1], w_only[3]])
    every = [t.detach().requires_grad_(True) for t in (x, *ws)]
    full = torch.autograd.grad(gated_feed_forward(*every).sum(), every)
    assert torch.equal(part[0], full[1]) and torch.equal(part[1], full[3])
    # against differences, first and second order
    step = [_rand(gen, *t.shape).to(device) for t in every]
    ct = _rand(gen, 3, 4, 6).to(device)

    def gradient(eps, create_graph=False):
        t = [(a + eps * d).detach().requires_grad_(True) for a, d in zip((x, *ws), step)]
        y = (gated_feed_forward(*t) * ct).sum()
        return t, y, torch.autograd.grad(y, t, create_graph=create_graph)
    eps = 2.0 ** -7
    t, _, grads = gradient(0.0, True)
    along = sum((g * d).sum() for g, d in zip(grads, step))
    up, down = gradient(eps), gradient(-eps)
    diff = (float(up[1]) - float(down[1])) / (2 * eps)
    assert abs(diff - float(along)) <= 5e-3 * (1 + abs(diff))
    for s, a, b in zip(torch.autograd.grad(along, t), up[2], down[2]):
        want = (a - b) / (2 * eps)
        assert float((s - want).abs().max()) <= 2e-2 * (1 + float(want.abs().max()))


def test_gated_feed_forward_passes_on_what_is_not_finite(device):
    """A row with a NaN spoils its own results and the weights' gradients, no other row's."""
    from equitorch_amd.nn.functional import gated_feed_forward
    gen = torch.Generator().manual_seed(2)
    x = _rand(gen, 200, 48).to(device)
    ws = [_rand(gen, *s, std=0.2).to(device) for s in ((48, 80), (48, 80), (80, 40))]
    clean = gated_feed_forward(x, *ws)
    x[77, 5] = float("nan")
    out = gated_feed_forward(x, *ws)
    keep = torch.arange(200, device=device) != 77
    assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[77]).all()


def test_gated_feed_forward_refuses(device):
    from equitorch_amd.nn.functional import gated_feed_forward
    x, wg, wu, wd = (torch.zeros(*s, device=device) for s in ((3, 8), (8, 6), (8, 6), (6, 4)))
    for bad in ((x, wg, wu[:, :5], wd), (x[:, :7], wg, wu, wd), (x, wg, wu, wd[:5]), (x.double(), wg.double(), wu.double(), wd.double()),
                (x.bfloat16(), wg, wu, wd), (x.cpu(), wg, wu, wd), (x, wg[0], wu[0], wd), (x, wg[:, :0], wu[:, :0], wd[:0]),
                (x, wg, wu, wd, "relu")):
        with pytest.raises(CgtpError):
            gated_feed_forward(*bad)


def test_extension_and_ctypes_issue_the_same_launches(device):
    """With the C++ extension's autograd nodes and without it: the same bits, and a second order either way, also when nobody
    holds the plan any more."""
    from equitorch_amd import _shim
    from equitorch_amd.nn.functional import AttentionPlan, embedding, gated_feed_forward, segment_attention
    assert _shim.module() is not None, "the extension is not built"
    gen = torch.Generator().manual_seed(21)
    n = 60
    kind = torch.randint(0, 7, (n,), generator=gen).to(device)
    data = [_rand(gen, 7, 32), _rand(gen, n, 3), torch.rand(2, generator=gen), _rand(gen, 32, 40, std=0.2), _rand(gen, 32, 40, std=0.2),
            _rand(gen, 40, 32, std=0.2)]
    seen = []
    for use_shim in (True, False):
        saved = _shim._module
        if not use_shim:
            _shim._module = None
        try:
            t = [d.to(device).requires_grad_(True) for d in data]
            x = embedding(kind, t[0], 2.0)
            assert ("Cpp" in type(x.grad_fn).__name__) == use_shim
            h = x.view(n, 2, 16)
            y = segment_attention(h, h, h, AttentionPlan(torch.tensor([0, 25, n], device=device)), pos=t[1], slope=t[2], cap=5.0)
            y = gated_feed_forward(y.reshape(n, 32), *t[3:])
            energy = (y * y).sum()
            first = torch.autograd.grad(energy, t, retain_graph=True)
            forces = torch.autograd.grad(energy, t[1], create_graph=True)[0]
            second = torch.autograd.grad((forces * forces).sum(), t)
            with torch.no_grad():
                again = gated_feed_forward(y.detach(), *t[3:])
        finally:
            _shim._module = saved
        seen.append([y, *first, again, forces, *second])
    for a, b in zip(seen[0][:-7], seen[1][:-7]):
        assert torch.equal(a, b)
    for a, b in zip(seen[0][-7:], seen[1][-7:]):            # tensor expressions: sums of the library's own order
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5 * float(b.abs().max()))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,c,h,co,activation", [(17001, 35, 130, 21, "silu"), (2100, 130, 1003, 67, "gelu"),
                                                    (33001, 9, 15, 13, "sigmoid"), (4001, 64, 520, 33, "silu")])
def test_gated_feed_forward_of_many_odd_rows(device, dtype, rows, c, h, co, activation):
    """Rows that are not whole aligned groups in a call large enough that they are copied first."""
    test_gated_feed_forward(device, dtype, rows, c, h, co, activation)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_gated_feed_forward_of_many_odd_rows_passes_on_what_is_not_finite(device, value):
    from equitorch_amd.nn.functional import gated_feed_forward
    gen = torch.Generator().manual_seed(3)
    x = _rand(gen, 9000, 31).to(device)
    ws = [_rand(gen, *s, std=0.2).to(device) for s in ((31, 250), (31, 250), (250, 30))]
    clean = gated_feed_forward(x, *ws)
    x[777, 30] = value
    out = gated_feed_forward(x, *ws)
    keep = torch.arange(9000, device=device) != 777
    assert torch.equal(out[keep], clean[keep]) and not torch.isfinite(out[777]).any()


def test_gated_feed_forward_at_unaligned_addresses(device):
    """The same numbers at addresses that are multiples of an element only, and in place of aligned ones."""
    from equitorch_amd.nn.functional import gated_feed_forward
    gen = torch.Generator().manual_seed(4)
    shapes = ((8192, 32), (32, 256), (32, 256), (256, 32))
    data = [_rand(gen, *s, dtype=BF16, std=0.3).to(device) for s in shapes]
    loose = [torch.empty(t.numel() + 1, dtype=BF16, device=device)[1:].view(t.shape).copy_(t) for t in data]
    results = []
    for given in (data, loose):
        leaves = [t.detach().requires_grad_(True) for t in given]
        out = gated_feed_forward(*leaves)
        results.append((out, *torch.autograd.grad(out.float().sum(), leaves)))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, F64, BF16])
@pytest.mark.parametrize("rows,kinds,channels", [(1, 9000, 5), (64, 1, 70), (200, 40, 513), (255, 7, 33), (256, 300, 8), (257, 5000, 200)])
def test_embedding_of_few_rows(device, dtype, rows, kinds, channels):
    """Where the gradient takes one launch, and just beyond: many rows of one kind, and a table much larger than the rows."""
    test_embedding(device, dtype, rows, kinds, channels)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,biased,cap", [
    ("short", 8, 8, 16, True, 0.0), ("short", 8, 4, 128, True, 0.0), ("short", 4, 4, 96, True, 5.0), ("short", 2, 2, 64, False, 0.0),
    ("odd", 4, 4, 32, True, 4.0), ("odd", 4, 1, 64, False, 0.0), ("odd", 2, 2, 128, True, 0.0), ("long", 2, 1, 72, True, 3.0),
    ("long", 2, 2, 128, False, 0.0), ("few_keys", 4, 2, 24, True, 0.0), ("mixed", 3, 3, 96, True, 6.0), ("mixed", 4, 4, 8, False, 0.0)])
def test_attention_as_in_a_large_batch(device, monkeypatch, dtype, lengths, heads, kv_heads, dim, biased, cap):
    """The tiles that a batch gets which fills the GPU: a wavefront for each, or four for 128 rows, and long pieces."""
    from equitorch_amd.nn.functional import attention
    monkeypatch.setattr(attention, "_SMALL", 0)
    test_attention(device, dtype, lengths, heads, kv_heads, dim, biased, cap)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("scale,cap", [(1.0, 1e-5), (0.125, 1e-6), (0.125, 1e-9), (1.0, 1e-30), (1.0, 1e-44), (1.0, 1e-60), (1e-3, 1e-6),
                                       (64.0, 1e-3), (1.0, 1e25), (1.0, 3e38), (1.0, 1e300), (0.0, 5.0)])
def test_attention_caps_of_every_size(device, dtype, scale, cap):
    """Scores within 1e-3 of one another at most, or as good as uncapped, in lengths that leave rows and keys of a tile empty."""
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    gen = torch.Generator().manual_seed(31)
    lengths, heads, dim = [1, 40, 33], 2, 24
    n = sum(lengths)
    q, k, v, ct = (_rand(gen, n, heads, dim, dtype=dtype) for _ in range(4))
    q[7] = 0.0                                             # scores of exactly zero
    val, mag, top = _reference(q, k, v, lengths, lengths, None, None, None, scale, cap, ct)
    plan = AttentionPlan(torch.tensor([0] + lengths, device=device).cumsum(0))
    leaves = [t.to(device).requires_grad_(True) for t in (q, k, v)]
    out = segment_attention(*leaves, plan, cap=cap, scale=scale)
    grads = torch.autograd.grad(out, leaves, ct.to(device))
    # as for other caps (test_attention); `top` bounds the products, not the scores, where these are within the cap
    unit = 4 * EPS[dtype] + EPS[F32] * (32 + dim + 16 * top) if dtype != F32 else EPS[F32] * (32 + dim + 16 * top)
    for name, got in zip(("out", "q", "k", "v"), (out, *grads)):
        _within(got, val[name], EPS[dtype] * val[name].abs() + unit * mag[name] + 64 * TINY[dtype], name)


def _attention_of_one_structure(q, k, v, ct, scale):
    """Result and gradients in 64 bits, one head after the other."""
    got = [torch.zeros_like(t) for t in (q, q, k, v)]
    for h in range(q.shape[1]):
        p = torch.softmax(q[:, h] @ k[:, h].T * scale, 1)
        dp = ct[:, h] @ v[:, h].T
        got[0][:, h], got[3][:, h] = p @ v[:, h], p.T @ ct[:, h]
        ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
        got[1][:, h], got[2][:, h] = ds @ k[:, h], ds.T @ q[:, h]
    return got


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("n_q,n_k,heads,dim,size,scale", [
    (4000, 4000, 1, 64, 1e-3, None), (4000, 4000, 1, 64, 1.0, None), (4000, 4000, 1, 64, 1e4, None), (16, 100003, 2, 32, 1e4, None),
    (1, 200003, 2, 16, 1e4, None), (300, 7001, 2, 96, 1e-2, None), (4, 5, 2, 128, 3e4, 2.0 ** -9), (6, 4, 1, 128, 3e4, 2.0 ** -9)])
def test_attention_fp16_gradients_of_any_size(device, monkeypatch, wide, n_q, n_k, heads, dim, size, scale):
    """Probabilities below fp16's normal range, and gradients of the scores below or beyond it where the results are within.  Each term of a
    sum is rounded by 2^-11 at most, in either direction, and so is the result: of its norm 2^-10 together, and half a
    subnormal step for each element."""
    from equitorch_amd.nn.functional import AttentionPlan, attention, segment_attention
    if not wide:
        monkeypatch.setattr(attention, "_SMALL", 0)
    gen = torch.Generator(device=device).manual_seed(41)
    draw = lambda n: torch.randn(n, heads, dim, generator=gen, device=device)
    q, k, v, ct = draw(n_q), draw(n_k), draw(n_k), draw(n_q).clamp(-1, 1) * size
    q, k, v, ct = (t.half() for t in (q, k, v, ct))
    plan = AttentionPlan(torch.tensor([0, n_q], device=device), torch.tensor([0, n_k], device=device))
    scale = dim ** -0.5 if scale is None else scale
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = segment_attention(*leaves, plan, scale=scale)
    grads = torch.autograd.grad(out, leaves, ct)
    want = _attention_of_one_structure(*(t.double() for t in (q, k, v, ct)), scale)
    for name, a, b in zip(("out", "q", "k", "v"), (out, *grads), want):
        err, most = float((a.double() - b).norm()), 2.0 ** -10 * float(b.norm()) + 2.0 ** -25 * b.numel() ** 0.5
        assert err <= most, f"{name}: {err:.3e} beyond {most:.3e}"


def test_attention_fp16_gradients_of_rows_of_different_size(device):
    """A column's factor is its own, falls as larger gradients come, and zeros, infinities and NaN stay theirs."""
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    gen = torch.Generator(device=device).manual_seed(42)
    n, dim = 600, 32
    q, k, v, ct = (torch.randn(n, 1, dim, generator=gen, device=device) for _ in range(4))
    ct = ct * torch.logspace(-6, 3, n, device=device)[:, None, None]
    ct[100:140] = 0.0
    q, k, v, ct = (t.half() for t in (q, k, v, ct))
    plan = AttentionPlan(torch.tensor([0, n], device=device))

    def gradients(ct):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(segment_attention(*leaves, plan), leaves, ct)
    got = gradients(ct)
    want = _attention_of_one_structure(*(t.double() for t in (q, k, v, ct)), dim ** -0.5)[1:]
    for row in range(n):                                   # dq: each row by its own size
        err, most = float((got[0][row].double() - want[0][row]).norm()), 2.0 ** -9 * float(want[0][row].norm()) + 2.0 ** -24 * dim ** 0.5
        assert err <= most, f"row {row}: {err:.3e} beyond {most:.3e}"
    assert torch.equal(got[0][100:140], torch.zeros_like(got[0][100:140]))
    for a, b in zip(got[1:], want[1:]):
        assert float((a.double() - b).norm()) <= 2.0 ** -10 * float(b.norm())
    ct[300] = float("inf")
    bad = gradients(ct)
    keep = torch.arange(n, device=device) != 300
    assert torch.equal(bad[0][keep], got[0][keep]) and not torch.isfinite(bad[0][300]).any()
    assert not torch.isfinite(bad[1]).any() and not torch.isfinite(bad[2]).any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("small", [256, 0])
@pytest.mark.parametrize("readout", [False, True])
def test_attention_nodes_beyond_any_distance(device, monkeypatch, dtype, small, readout):
    """A node so far off that its squared distance is infinite in fp32 takes no part: results and gradients stay finite."""
    from equitorch_amd.nn.functional import AttentionPlan, attention, segment_attention
    monkeypatch.setattr(attention, "_SMALL", small)
    gen = torch.Generator().manual_seed(51)
    len_k, heads, dim = [40, 150], 2, 16
    len_q = [2, 3] if readout else len_k
    nq, nk = sum(len_q), sum(len_k)
    q, ct = (_rand(gen, nq, heads, dim, dtype=dtype) for _ in range(2))
    k, v = (_rand(gen, nk, heads, dim, dtype=dtype) for _ in range(2))
    pos_k, slope = _rand(gen, nk, 3), torch.rand(heads, generator=gen) + 0.1
    pos_k[[3, 39, 77]] = torch.tensor([[1e20, 0.0, 0.0], [0.0, -3e19, 1e19], [2e25, 2e25, 2e25]])
    pos = _rand(gen, nq, 3) if readout else pos_k
    val, mag, top = _reference(q, k, v, len_q, len_k, pos, pos_k, slope, dim ** -0.5, 0.0, ct)
    ptr = lambda n: torch.tensor([0] + n, device=device).cumsum(0)
    plan = AttentionPlan(ptr(len_q), ptr(len_k)) if readout else AttentionPlan(ptr(len_k))
    leaves = [t.to(device).requires_grad_(True) for t in (q, k, v, pos, slope)]
    more = [pos_k.to(device).requires_grad_(True)] if readout else []
    out = segment_attention(*leaves[:3], plan, pos=leaves[3], slope=leaves[4], pos_k=more[0] if more else None)
    grads = torch.autograd.grad(out, leaves + more, ct.to(device))
    if not readout:
        val["pos"], mag["pos"] = val["pos"] + val["pos_k"], mag["pos"] + mag["pos_k"]
    # as in test_attention, for the scores of nodes that take part: 40 at most
    unit = 4 * EPS[dtype] + EPS[F32] * (32 + dim + 16 * 40) if dtype != F32 else EPS[F32] * (32 + dim + 16 * 40)
    for name, got in zip(("out", "q", "k", "v", "pos", "slope", "pos_k"), (out, *grads)):
        own_type = EPS[F32] if name in ("pos", "pos_k", "slope") else EPS[dtype]
        _within(got, val[name], own_type * val[name].abs() + unit * mag[name] + 64 * TINY[dtype], name)


def test_attention_plan_does_not_grow_with_scales_and_caps(device):
    """A scale or a cap that changes every step leaves nothing behind on a lasting plan; the second order knows it all the same."""
    from equitorch_amd import _shim
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    gen = torch.Generator().manual_seed(61)
    plan = AttentionPlan(torch.tensor([0, 12, 30], device=device))
    data = [_rand(gen, 30, 2, 8) for _ in range(4)]
    seen = []
    for step in range(5):
        scale, cap = 0.3 + 0.1 * step, 2.0 + step
        q, k, v, ct = (t.to(device).requires_grad_(True) for t in data)
        out = segment_attention(q, k, v, plan, cap=cap, scale=scale)
        (gq,) = torch.autograd.grad(out, q, ct, create_graph=True)
        (gk,) = torch.autograd.grad(gq.square().sum(), k)
        wide = [t.double().requires_grad_(True) for t in data]
        want = torch.cat([torch.einsum("hij,jhd->ihd", torch.softmax(cap * torch.tanh(torch.einsum("ihd,jhd->hij", wide[0][s], wide[1][s])
                                                                                      * scale / cap), -1), wide[2][s])
                          for s in (slice(0, 12), slice(12, 30))])
        (rq,) = torch.autograd.grad(want, wide[0], wide[3], create_graph=True)
        (rk,) = torch.autograd.grad(rq.square().sum(), wide[1])
        for a, b in ((out, want), (gq, rq), (gk, rk)):     # fp32, sums of some hundred terms
            assert float((a.detach().cpu().double() - b.detach()).abs().max()) <= 1e-4 * max(1.0, float(b.abs().max()))
        seen.append(len(plan._tables) + len(plan._handles))
    assert _shim.module() is not None and seen == [2] * 5


@pytest.mark.parametrize("use_extension", [True, False])
def test_attention_plan_dropped_while_another_stream_reads_it(device, monkeypatch, use_extension):
    """The tables' memory is not handed out again before the work that another stream has queued with them is done."""
    from equitorch_amd import _shim
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    if not use_extension:
        monkeypatch.setattr(_shim, "_module", None)
    n, count = 21, 4000                                    # tables of a size of their own, 128 kB
    ptr = torch.arange(count + 1, device=device) * n
    q = torch.randn(n * count, 1, 16, device=device)
    want = segment_attention(q, q, q, AttentionPlan(ptr))
    plan = AttentionPlan(ptr)
    table = plan.tables(1, 1).q_items
    place, size = table.data_ptr(), table.numel() * table.element_size()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)                     # a bounded wait, some 50 ms
        out = segment_attention(q, q, q, plan)
    del plan, table
    ours = [torch.empty(size, dtype=torch.uint8, device=device) for _ in range(20)]
    assert not side.query(), "the other stream was done too early to tell"
    assert place not in {t.data_ptr() for t in ours}
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_gated_feed_forward_of_millions_of_wide_rows(device):
    """More rows than fit 2^31 elements of what is kept: rows here and there against 64 bits."""
    from equitorch_amd.nn.functional import gated_feed_forward
    gen = torch.Generator(device=device).manual_seed(71)
    rows, c, hidden = 2200001, 8, 8192
    draw = lambda *s, std=1.0: (torch.randn(*s, generator=gen, device=device) * std).bfloat16()
    x, wg, wu, wd = draw(rows, c), draw(c, hidden, std=c ** -0.5), draw(c, hidden, std=c ** -0.5), draw(hidden, c, std=hidden ** -0.5)
    with torch.no_grad():
        out = gated_feed_forward(x, wg, wu, wd)
    at = torch.cat([torch.randint(0, rows, (60,), generator=gen, device=device), torch.tensor([0, 262143, 262144, rows - 1], device=device)])
    g, u, w = (t.double() for t in (x[at].double() @ wg.double(), x[at].double() @ wu.double(), wd))
    mid = g * torch.sigmoid(g) * u
    # the products' sums in fp32, mid and the result rounded to bf16
    bound = EPS[BF16] * ((mid @ w).abs() + 1.1 * mid.abs() @ w.abs()) + 1e-5
    _within(out[at], (mid @ w).cpu(), bound.cpu(), "out")


def test_gated_feed_forward_of_weights_beyond_31_bits(device):
    """Weights with more than 2^31 elements together: results, and their gradients at places here and there, against 64 bits."""
    from equitorch_amd.nn.functional import gated_feed_forward
    gen = torch.Generator(device=device).manual_seed(72)
    rows, c, hidden = 5, 12000, 65000
    draw = lambda *s, std=1.0: (torch.randn(*s, generator=gen, device=device) * std).bfloat16()
    t = [draw(rows, c), draw(c, hidden, std=c ** -0.5), draw(c, hidden, std=c ** -0.5), draw(hidden, c, std=hidden ** -0.5)]
    t = [a.requires_grad_(True) for a in t]
    ct = draw(rows, c)
    out = gated_feed_forward(*t)
    got = torch.autograd.grad(out, t, ct)
    x, wg, wu, wd = (a.detach() for a in t)
    want, size, gx, size_x = (torch.zeros(rows, c, dtype=F64, device=device) for _ in range(4))
    cols = torch.tensor([0, 1, 32767, 32768, 64999], device=device)
    xd, cd = x.double(), ct.double()
    for h in range(0, hidden, 5000):
        s = slice(h, h + 5000)
        g, u, gm = xd @ wg[:, s].double(), xd @ wu[:, s].double(), cd @ wd[s].double().T
        sig = torch.sigmoid(g)
        mid, dg, du = g * sig * u, gm * u * (sig + g * sig * (1 - sig)), gm * g * sig
        want += mid @ wd[s].double()
        size += mid.abs() @ wd[s].double().abs()
        gx += dg @ wg[:, s].double().T + du @ wu[:, s].double().T
        # dg and du are rounded, as are g and u that they are formed from: four roundings of terms of this size
        size_x += (gm * u).abs() @ wg[:, s].double().abs().T + (gm * g).abs() @ wu[:, s].double().abs().T
        here = cols[(cols >= h) & (cols < h + 5000)] - h
        for name, a, b, m in (("w_gate", got[1][:, here + h], xd.T @ dg[:, here], xd.abs().T @ (gm * u).abs()[:, here]),
                              ("w_up", got[2][:, here + h], xd.T @ du[:, here], xd.abs().T @ (gm * g).abs()[:, here]),
                              ("w_down", got[3][here + h], mid[:, here].T @ cd, mid.abs()[:, here].T @ cd.abs())):
            _within(a, b.cpu(), (EPS[BF16] * (b.abs() + 6 * m) + 1e-4 * m).cpu(), name)
    _within(out, want.cpu(), (EPS[BF16] * (want.abs() + 1.1 * size) + 1e-4 * size).cpu(), "out")
    _within(got[0], gx.cpu(), (EPS[BF16] * (gx.abs() + 6 * size_x) + 1e-4 * size_x).cpu(), "x")


@pytest.mark.parametrize("use_extension", [True, False])
@pytest.mark.parametrize("operator", ["embedding", "attention", "feed_forward"])
def test_tangents_are_refused_not_dropped(device, monkeypatch, use_extension, operator):
    """Forward-mode differentiation is not served: an operand with a tangent raises, one without gives the usual result."""
    import torch.autograd.forward_ad as forward_ad
    from equitorch_amd import _shim
    from equitorch_amd.nn.functional import AttentionPlan, embedding, gated_feed_forward, segment_attention
    if not use_extension:
        monkeypatch.setattr(_shim, "_module", None)
    gen = torch.Generator().manual_seed(81)
    plan, kind = AttentionPlan(torch.tensor([0, 9], device=device)), torch.arange(9, device=device)
    x, w = _rand(gen, 9, 8).to(device), _rand(gen, 8, 8).to(device)
    run = {"embedding": lambda x: embedding(kind, x), "feed_forward": lambda x: gated_feed_forward(x, w, w, w),
           "attention": lambda x: segment_attention(*[x.view(9, 2, 4)] * 3, plan)}[operator]
    want = run(x)
    with forward_ad.dual_level():
        assert torch.equal(run(x), want)
        with pytest.raises((RuntimeError, NotImplementedError)):
            run(forward_ad.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError)):
            run(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_operands_of_different_types_under_autocast(device, dtype):
    """16-bit features and fp32 weights: as with every operand rounded to autocast's type; gradients in the operands' own types.
    Without autocast they are refused."""
    from equitorch_amd.nn import GatedFeedForward, SegmentAttention
    from equitorch_amd.nn.functional import AttentionPlan, gated_feed_forward, segment_attention
    gen = torch.Generator().manual_seed(91)
    x = _rand(gen, 30, 16, dtype=dtype).to(device)
    ws = [_rand(gen, *s, std=0.3).to(device).requires_grad_(True) for s in ((16, 24), (16, 24), (24, 16))]
    rounded = [w.detach().to(dtype).requires_grad_(True) for w in ws]
    want = gated_feed_forward(x, *rounded)
    grads = torch.autograd.grad(want.float().sum(), rounded)
    with torch.autocast("cuda", dtype=dtype):
        out = gated_feed_forward(x, *ws)
    got = torch.autograd.grad(out.float().sum(), ws)
    assert out.dtype == dtype and torch.equal(out, want)
    for a, b in zip(got, grads):
        assert a.dtype == F32 and torch.equal(a, b.float())
    plan = AttentionPlan(torch.tensor([0, 11, 30], device=device))
    q = x.view(30, 2, 8)
    with torch.autocast("cuda", dtype=dtype):
        assert torch.equal(segment_attention(q, q.float(), q, plan), segment_attention(q, q, q, plan))
        for bad in ((x.double(), *ws), (x, ws[0].double(), *ws[1:])):
            with pytest.raises(CgtpError):
                gated_feed_forward(*bad)
        attention, block = SegmentAttention(16, 2).to(device), GatedFeedForward(16, 24).to(device)
        y = block(attention(x, plan, torch.zeros(30, 3, device=device)))
    assert y.dtype == dtype and torch.isfinite(y).all()
    with pytest.raises(CgtpError):
        gated_feed_forward(x, *ws)
    with pytest.raises(CgtpError):
        segment_attention(q, q.float(), q, plan)


LENGTHS["one long among many short"] = ([1] * 200, [5, 0, 33, 64] * 25 + [30011] + [7] * 99)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,biased,cap", [(8, 8, 32, True, 0.0), (4, 1, 20, False, 3.0)])
def test_attention_of_one_long_structure_among_many(device, dtype, heads, kv_heads, dim, biased, cap):
    """Where the keys of one structure are cut and all others' are not."""
    test_attention(device, dtype, "one long among many short", heads, kv_heads, dim, biased, cap)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("keys", [1, 40, 700])
@pytest.mark.parametrize("biased", [False, True])
def test_attention_gradients_of_a_row_of_nothing(device, dtype, keys, biased):
    """Every score of a structure -inf: its results and gradients are zeros, in one piece or several; another structure's are as without
    it."""
    from equitorch_amd.nn.functional import AttentionPlan, segment_attention
    gen = torch.Generator().manual_seed(101)
    n = keys + 9
    q, k, v, ct = (_rand(gen, n, 2, 16, dtype=dtype).abs().to(device) for _ in range(4))
    pos, slope = _rand(gen, n, 3).to(device), torch.rand(2, generator=gen).to(device)
    k[:keys] = -torch.inf

    def run(rows, lengths):
        t = [a[rows].clone().requires_grad_(True) for a in (q, k, v, pos)]
        out = segment_attention(*t[:3], AttentionPlan(torch.tensor([0] + lengths, device=device).cumsum(0)),
                                pos=t[3] if biased else None, slope=slope if biased else None)
        return (out, *torch.autograd.grad(out, t if biased else t[:3], ct[rows]))
    both, alone = run(slice(0, n), [keys, 9]), run(slice(keys, n), [9])
    for a, b in zip(both, alone):
        assert torch.equal(a[:keys], torch.zeros_like(a[:keys]))
        assert float((a[keys:].float() - b.float()).abs().max()) <= 2 * EPS[dtype] * max(1.0, float(b.float().abs().max()))


@pytest.mark.parametrize("use_extension", [True, False])
@pytest.mark.parametrize("operator", ["embedding", "attention", "feed_forward"])
def test_batched_gradients_are_refused(device, monkeypatch, use_extension, operator):
    """A gradient that a transform has batched has no memory of its own to read: an error, no launch."""
    from equitorch_amd import _shim
    from equitorch_amd.nn.functional import AttentionPlan, embedding, gated_feed_forward, segment_attention
    if not use_extension:
        monkeypatch.setattr(_shim, "_module", None)
    gen = torch.Generator().manual_seed(111)
    plan, kind = AttentionPlan(torch.tensor([0, 9], device=device)), torch.arange(9, device=device)
    x, w = _rand(gen, 9, 8).to(device).requires_grad_(True), _rand(gen, 8, 8).to(device)
    out = {"embedding": lambda: embedding(kind, x), "feed_forward": lambda: gated_feed_forward(x, w, w, w),
           "attention": lambda: segment_attention(*[x.view(9, 2, 4)] * 3, plan).reshape(9, 8)}[operator]()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, x, torch.ones(3, 9, 8, device=device), is_grads_batched=True)
    (g,) = torch.autograd.grad(out, x, torch.ones(9, 8, device=device))
    assert torch.isfinite(g).all()
