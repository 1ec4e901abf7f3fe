"""Cross entropy over kinds against its definition in 64 bits.

Tolerances are bounds on rounding, element by element: the result's own rounding, plus the roundings of what is held in 32
bits or in the operands' type times the magnitudes that enter the element."""
import pytest
import torch

from equitorch_amd._lib import CgtpError
from helpers import stable_seed

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
EPS = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
U = 2.0 ** -24


def _rand(gen, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=gen, dtype=F64) * std).to(dtype)


def _within(got, want, bound, what):
    got, want = got.detach().to(want.device).double(), want.double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} vs {tuple(want.shape)}"
    excess = ((got - want).abs() - bound).max() if want.numel() else torch.tensor(-1.0)
    assert float(excess) <= 0 and torch.isfinite(got).all(), f"{what}: {float(excess):.3e} over the bound"


def _check(got, x, table, kind, scale, cap, g, dtype):
    """(loss, grad_x, grad_table) against the formulas, row by row those that have a kind."""
    n, c = x.shape
    k = table.shape[0]
    asked = ((kind >= 0) & (kind < k)).nonzero()[:, 0]
    y = kind[asked]
    w, xs, gs = table.double(), x[asked].double(), g[asked].double()[:, None]
    raw = xs @ w.T * scale
    err = (c + 4) * U * (xs.abs() @ w.abs().T) * abs(scale)              # of a product over C and the scale
    th = torch.tanh(raw / cap) if cap else torch.zeros_like(raw)
    z = cap * th if cap else raw
    if cap:
        # a hyperbolic tangent to some roundings of itself, or of 1 in a block with large ones: 1 - e and 1 + e, the reciprocal and the products
        err = err + 10 * U * z.abs() + (3 * U * cap if raw.numel() and float((raw / cap).abs().max()) > 0.25 else 0.0)
    err = err + 4 * U * z.abs().amax(1, keepdim=True)                    # to the base 2, less the maximum
    most = err.amax(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    delta = most + (k / 4 + 40) * U                                      # of lse: its terms' errors, and a sum in chains of K / 4
    loss = torch.zeros(n, dtype=F64, device=x.device)
    bound = torch.zeros_like(loss)
    loss[asked] = (lse - z.gather(1, y[:, None]))[:, 0]
    bound[asked] = (delta + err.gather(1, y[:, None]) + 4 * U * (lse.abs() + loss[asked][:, None].abs()))[:, 0]
    _within(got[0], loss, bound, "loss")
    if got[1] is None and got[2] is None:
        return
    one = torch.zeros_like(z).scatter_(1, y[:, None], 1.0)
    p = (z - lse).exp()
    slope = 1 - th * th
    dz = (p - one) * slope
    # the slope 1 - t^2 has twice t's eleven roundings and its own
    if cap:
        err = err + 12 * U * cap        # the gradients' logits have the tangent from one exponential: some roundings of 1
    off = 2 * p * (err + delta + 2 * U * (z - lse).abs()) + 2 * U * one + (24 * U if cap else 0) * (p + one)
    off = off + EPS[dtype] * (dz.abs() + off) + (2.0 ** -40 if dtype == F16 else 2.0 ** -120)
    if got[1] is not None:
        want, size = torch.zeros(n, c, dtype=F64, device=x.device), torch.zeros(n, c, dtype=F64, device=x.device)
        want[asked] = gs * scale * (dz @ w)
        size[asked] = gs.abs() * abs(scale) * ((off + (k + 4) * U * dz.abs()) @ w.abs())
        _within(got[1], want, EPS[dtype] * (want.abs() + size) + size + (2.0 ** -25 if dtype == F16 else 0), "grad_x")
    if got[2] is not None:
        top = float(gs.abs().max()) if len(asked) else 0.0
        xg, rounding = gs * xs, EPS[dtype] * (gs * xs).abs() + (top * 2.0 ** -25 if dtype == F16 else 0)
        want = scale * (dz.T @ xg)
        size = abs(scale) * ((off + (n + 8) * U * dz.abs()).T @ (xg.abs() + rounding) + dz.abs().T @ rounding)
        _within(got[2], want, EPS[dtype] * (want.abs() + size) + size + (2.0 ** -25 if dtype == F16 else 0), "grad_table")


def _inputs(seed, rows, kinds, channels, dtype, masked):
    gen = torch.Generator().manual_seed(seed)
    x, table = _rand(gen, rows, channels, dtype=dtype), _rand(gen, kinds, channels, dtype=dtype)
    kind = torch.randint(0, kinds, (rows,), generator=gen)
    hidden = torch.rand(rows, generator=gen) < masked
    kind[hidden] = torch.where(torch.arange(int(hidden.sum())) % 2 == 0, -1, kinds)
    x[hidden] = float("nan")                                             # what is not asked for is not read
    g = _rand(gen, rows) if rows % 2 else torch.full((rows,), 1.0 / rows)
    g[hidden] = float("nan")
    return x, table, kind, g


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,kinds,channels,masked,cap", [
    (1, 1, 1, 0.0, None), (1, 2, 8, 0.0, None), (30, 100, 64, 0.0, None), (31, 100, 64, 0.3, 5.0), (129, 257, 40, 0.0, 20.0), (64, 128, 32, 0.0, None),
    (65, 129, 33, 0.5, None), (301, 1000, 33, 0.85, 3.0), (1001, 3000, 100, 0.1, None), (130, 129, 512, 0.0, None), (5, 20011, 16, 0.0, None),
    (2001, 10, 7, 0.7, None), (3, 40, 1003, 0.0, 30.0), (70, 5, 20, 1.0, None)])
def test_kind_cross_entropy(device, dtype, rows, kinds, channels, masked, cap):
    from equitorch_amd.nn.functional import kind_cross_entropy
    x, table, kind, g = _inputs(stable_seed(rows, kinds, channels), rows, kinds, channels, dtype, masked)
    scale = 1.5 * channels ** -0.5
    leaves = [t.to(device).requires_grad_(True) for t in (x, table)]
    loss = kind_cross_entropy(*leaves, kind.to(device), scale, cap)
    assert loss.dtype == F32 and loss.shape == (rows,)
    grads = torch.autograd.grad(loss, leaves, g.to(device), retain_graph=True)
    _check((loss, *grads), x, table, kind, scale, cap, g, dtype)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(loss, leaves, g.to(device))))
    with torch.no_grad():
        assert torch.equal(kind_cross_entropy(*leaves, kind.to(device), scale, cap), loss)


@pytest.mark.parametrize("rows,kinds,channels,dtype", [(40003, 10007, 16, BF16), (35001, 5003, 8, F32), (33001, 9001, 264, F16), (140001, 300, 8, F16),
                                                       (300, 300011, 8, F16), (20011, 130, 100, BF16), (300001, 20, 8, F32), (270001, 140, 24, F16)])
def test_pieces(device, rows, kinds, channels, dtype):
    """More rows, or kinds, or both, than the backward takes at a time; many of one and few of the other."""
    from equitorch_amd.nn.functional import kind_cross_entropy
    x, table, kind, g = (t.to(device) for t in _inputs(stable_seed(rows, kinds), rows, kinds, channels, dtype, 0.02))
    leaves = [t.clone().requires_grad_(True) for t in (x, table)]
    loss = kind_cross_entropy(*leaves, kind, 0.3)
    grads = torch.autograd.grad(loss, leaves, g)
    _check((loss, *grads), x, table, kind, 0.3, None, g, dtype)


def test_one_gradient_at_a_time(device):
    from equitorch_amd.nn.functional import kind_cross_entropy
    x, table, kind, g = _inputs(3, 301, 700, 24, BF16, 0.2)
    leaves = [t.to(device).requires_grad_(True) for t in (x, table)]
    both = torch.autograd.grad(kind_cross_entropy(*leaves, kind.to(device)), leaves, g.to(device))
    for i in (0, 1):
        one = [t.detach().requires_grad_(i == j) for j, t in enumerate(leaves)]
        (grad,) = torch.autograd.grad(kind_cross_entropy(*one, kind.to(device)), one[i], g.to(device))
        assert torch.equal(grad, both[i])


def test_large_logits(device):
    """Probabilities of one and of nothing: no overflow, no NaN."""
    from equitorch_amd.nn.functional import kind_cross_entropy
    for dtype in (F32, BF16, F16):
        x, table, kind, g = _inputs(4, 201, 333, 16, dtype, 0.0)
        leaves = [t.to(device).requires_grad_(True) for t in (x, table)]
        loss = kind_cross_entropy(*leaves, kind.to(device), 300.0)
        _check((loss, *torch.autograd.grad(loss, leaves, g.to(device))), x, table, kind, 300.0, None, g, dtype)
        loss = kind_cross_entropy(*leaves, kind.to(device), 1e4, 2.0)
        assert torch.isfinite(loss).all() and all(torch.isfinite(t).all() for t in torch.autograd.grad(loss, leaves, g.to(device)))


@pytest.mark.parametrize("scale,cap", [(-0.4, None), (-0.4, 2.0), (0.0, None), (0.0, 2.0)])
def test_scales_of_either_sign(device, scale, cap):
    from equitorch_amd.nn.functional import kind_cross_entropy
    for dtype in (F32, BF16):
        x, table, kind, g = _inputs(11, 77, 150, 24, dtype, 0.1)
        leaves = [t.to(device).requires_grad_(True) for t in (x, table)]
        loss = kind_cross_entropy(*leaves, kind.to(device), scale, cap)
        _check((loss, *torch.autograd.grad(loss, leaves, g.to(device))), x, table, kind, scale, cap, g, dtype)


def test_what_is_not_finite_stays_in_its_row(device):
    """An infinity in a row that is asked for makes its loss and its gradient NaN and, through the table's gradient, all of that; the other
    rows' losses and gradients are theirs."""
    from equitorch_amd.nn.functional import kind_cross_entropy
    for dtype, channels in ((F32, 24), (BF16, 24), (F16, 300)):
        x, table, kind, _ = _inputs(12, 90, 70, channels, dtype, 0.0)
        good = kind_cross_entropy(x.to(device), table.to(device), kind.to(device), 0.1)
        x[17, 3] = float("inf")
        leaves = [t.to(device).requires_grad_(True) for t in (x, table)]
        loss = kind_cross_entropy(*leaves, kind.to(device), 0.1)
        others = torch.arange(90, device=device) != 17
        assert torch.isnan(loss[17]) and torch.equal(loss[others], good[others])
        gx, gw = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
        assert torch.isnan(gx[17]).any() and torch.isfinite(gx[others]).all() and torch.isnan(gw).any()


def test_batched_gradients_are_refused(device):
    from equitorch_amd.nn.functional import kind_cross_entropy
    x = torch.randn(5, 8, device=device, requires_grad=True)
    loss = kind_cross_entropy(x, torch.randn(7, 8, device=device), torch.arange(5, device=device))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, x, torch.ones(3, 5, device=device), is_grads_batched=True)


@pytest.mark.parametrize("n,k,c,cap", [(700, 900, 300, None), (130, 2001, 384, 3.0), (40, 5003, 512, None), (3000, 170, 449, None), (1, 129, 257, 2.0),
                                       (20000, 130, 390, None), (500, 33, 500, None)])
def test_gradients_of_more_than_256_channels(device, n, k, c, cap):
    from equitorch_amd.nn.functional import kind_cross_entropy
    for dtype, wanted in ((BF16, (True, True)), (F16, (True, True)), (BF16, (False, True)), (F16, (True, False))):
        x, table, kind, g = _inputs(stable_seed(n, k, c), n, k, c, dtype, 0.3)
        leaves = [t.to(device).requires_grad_(w) for t, w in zip((x, table), wanted)]
        loss = kind_cross_entropy(*leaves, kind.to(device), 0.06, cap)
        grads = iter(torch.autograd.grad(loss, [t for t in leaves if t.requires_grad], g.to(device)))
        got = [loss] + [next(grads) if w else None for w in wanted]
        if all(wanted):
            _check(got, x, table, kind, 0.06, cap, g, dtype)
            both = {dtype: got} if dtype == BF16 else {**both, dtype: got}
        else:                       # one alone: from another kernel or without the other's, of the same numbers
            _check((loss, None, None), x, table, kind, 0.06, cap, g, dtype)
            for one, two in zip(got[1:], both[dtype][1:]):
                assert one is None or float((one - two).abs().max()) <= 8 * EPS[dtype] * float(two.abs().max())


def test_rows_and_table_of_one_leaf(device):
    from equitorch_amd.nn.functional import kind_cross_entropy
    for dtype in (F32, BF16):
        table = _inputs(13, 5, 60, 40, dtype, 0.0)[1].to(device)
        kind, g = (torch.arange(60, device=device) + 7) % 61 - 1, torch.rand(60, device=device)
        one = table.clone().requires_grad_(True)
        two = [table.clone().requires_grad_(True) for _ in range(2)]
        got, = torch.autograd.grad(kind_cross_entropy(one, one, kind, 0.2), one, g)
        gx, gw = torch.autograd.grad(kind_cross_entropy(*two, kind, 0.2), two, g)
        assert torch.equal(got, gx + gw)


@pytest.mark.parametrize("dtype,k,c", [(BF16, (1 << 23) + 77, 256), (F32, (1 << 21) + 1011, 1024)])
def test_offsets_beyond_32_bits_in_the_table(device, dtype, k, c):
    from equitorch_amd.nn.functional import kind_cross_entropy
    n, gen = 20, torch.Generator(device=device).manual_seed(5)
    x = torch.randn(n, c, device=device, generator=gen).to(dtype)
    table = torch.randn(k, c, device=device, generator=gen, dtype=dtype)
    kind = k - 1 - 37 * torch.arange(n, device=device)
    kind[3], kind[4] = 0, -1
    g = torch.rand(n, device=device, generator=gen)
    leaves = [t.requires_grad_(True) for t in (x, table)]
    loss = kind_cross_entropy(*leaves, kind, 0.1)
    gx, gw = torch.autograd.grad(loss, leaves, g)
    x, table = x.detach(), table.detach()
    with torch.no_grad():
        # the logits in 64 bits, and what the gradients have of the rows near both ends of the table
        z = torch.cat([x.double() @ part.double().T for part in table.split(1 << 18)], 1) * 0.1
        p = (z - torch.logsumexp(z, 1, keepdim=True)).exp()
        asked = torch.arange(n, device=device) != 4
        want = (torch.logsumexp(z, 1) - z.gather(1, kind.clamp(min=0)[:, None])[:, 0]) * asked
        # of a logit: the product over C and the scale; of the sum's logarithm: chains of no more than all terms of a range
        err = (c + 8) * U * 0.1 * (x.double().norm(dim=1) * table[::997].double().norm(dim=1).max() * 1.2) + 8 * U * z.abs().amax(1)
        assert ((loss - want).abs() <= 2 * err + (k / 4 + 40) * U).all()
        p[torch.arange(n, device=device)[asked], kind[asked]] -= 1
        dz = p * (g * asked).double()[:, None] * 0.1
        size = dz.abs()
        off = 3 * EPS[dtype] + 4 * float(err.max()) + (k / 4 + 40) * U         # of dz, of x over the largest g, and of a product's result
        for rows in (slice(0, 300), slice(k - 1100, k)):
            _within(gw[rows], dz[:, rows].T @ x.double(), off * (size[:, rows].T @ x.double().abs()) + 2.0 ** -60, "grad table")
        want, bound = torch.zeros(n, c, dtype=F64, device=device), torch.zeros(n, c, dtype=F64, device=device)
        at = 0
        for part in table.split(1 << 18):
            d = dz[:, at:at + len(part)]
            want += d @ part.double()
            bound += d.abs() @ part.double().abs()
            at += len(part)
        _within(gx, want, (off + (k / 4 + 40) * U) * bound, "grad x")


def test_offsets_beyond_32_bits_in_the_rows(device):
    """Every row's results are those of the rows alone; the table's gradient has terms of the last ones only."""
    from equitorch_amd.nn.functional import kind_cross_entropy
    n, c, k, tail = (1 << 23) + 5003, 256, 40, 3000
    gen = torch.Generator(device=device).manual_seed(6)
    x = torch.randn(n, c, device=device, generator=gen, dtype=BF16)
    table = torch.randn(k, c, device=device, generator=gen, dtype=BF16).requires_grad_(True)
    kind = torch.randint(0, k, (n,), device=device, generator=gen)
    g = torch.zeros(n, device=device)
    g[-tail:] = torch.rand(tail, device=device, generator=gen)
    results = []
    for rows in (slice(None), slice(n - tail, None)):
        leaf = x[rows].detach().requires_grad_(True)
        loss = kind_cross_entropy(leaf, table, kind[rows], 0.1)
        gx, gw = torch.autograd.grad(loss, (leaf, table), g[rows])
        results.append((loss.detach()[-tail:].clone(), gx[-tail:].clone(), gw))
        if loss.numel() == n:
            assert not gx[:-tail].any()
    for a, b in zip(results[0][:2], results[1][:2]):
        assert torch.equal(a, b)
    # two sums of the same terms, of at most |x| 0.1 g each, in other orders, and each rounded once
    size = 0.1 * (g[-tail:, None] * x[-tail:].abs().float()).sum(0).double()
    gap = (results[0][2].double() - results[1][2].double()).abs()
    assert (gap <= 2 * 3000 * U * size + 2 * EPS[BF16] * results[1][2].double().abs()).all()


def test_small_incoming_gradients_in_fp16(device):
    """Gradients of one row and of the mean over many, whose products with probabilities are below fp16's range."""
    from equitorch_amd.nn.functional import kind_cross_entropy
    x, table, kind, g = _inputs(5, 201, 5000, 16, F16, 0.0)
    for size in (1e-3, 1.0):
        leaves = [t.to(device).requires_grad_(True) for t in (x, table)]
        weights = torch.full_like(g, size)
        weights[7] = size * 2.0 ** -12
        loss = kind_cross_entropy(*leaves, kind.to(device), 0.25)
        _check((loss, *torch.autograd.grad(loss, leaves, weights.to(device))), x, table, kind, 0.25, None, weights, F16)


def test_no_gradient_comes_in(device):
    from equitorch_amd.nn.functional import kind_cross_entropy
    x, table, kind, _ = _inputs(6, 77, 50, 16, F32, 0.1)
    leaves = [t.to(device).requires_grad_(True) for t in (x, table)]
    loss = kind_cross_entropy(*leaves, kind.to(device))
    for grad in torch.autograd.grad(loss, leaves, torch.zeros(77, device=device)):
        assert torch.equal(grad, torch.zeros_like(grad))


def test_shapes_strides_and_streams(device):
    from equitorch_amd.nn.functional import kind_cross_entropy
    gen = torch.Generator().manual_seed(7)
    x, table = _rand(gen, 4, 25, 19).to(device), _rand(gen, 60, 19).to(device)
    kind = torch.randint(-1, 60, (4, 25), generator=gen).to(device)
    want = kind_cross_entropy(x.reshape(100, 19), table, kind.reshape(100)).reshape(4, 25)
    assert torch.equal(kind_cross_entropy(x, table, kind), want)
    assert torch.equal(kind_cross_entropy(x.transpose(0, 1), table.T.contiguous().T, kind.T), want.T)
    loose = torch.empty(60 * 19 + 1, device=device)[1:].view(60, 19).copy_(table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kind_cross_entropy(x, loose, kind)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    assert torch.equal(kind_cross_entropy(x[0, 0], table, kind[0, 0]), want[0, 0])
    none = table.clone().requires_grad_(True)
    empty = kind_cross_entropy(x[:0], none, kind[:0])
    assert empty.shape == (0, 25)
    (grad,) = torch.autograd.grad(empty.sum(), none)
    assert torch.equal(grad, torch.zeros_like(grad))


def test_tied_to_an_embedding(device):
    """One table is looked up and scored against: its gradient is the sum of both."""
    from equitorch_amd.nn.functional import embedding, kind_cross_entropy
    gen = torch.Generator().manual_seed(8)
    table = _rand(gen, 30, 12).to(device).requires_grad_(True)
    seen, asked = (torch.randint(0, 30, (50,), generator=gen).to(device) for _ in range(2))
    (got,) = torch.autograd.grad(kind_cross_entropy(embedding(seen, table), table, asked, 0.5).mean(), table)
    wide = table.detach().double().requires_grad_(True)
    loss = torch.nn.functional.cross_entropy(wide[seen] @ wide.T * 0.5, asked)
    (want,) = torch.autograd.grad(loss, wide)
    _within(got, want, 1e-5 * want.abs().max(), "table")      # some hundred roundings of 2^-24 of the largest


def test_higher_order_and_differences(device):
    from equitorch_amd.nn.functional import kind_cross_entropy
    gen = torch.Generator().manual_seed(9)
    x, table = _rand(gen, 15, 9).to(device).requires_grad_(True), _rand(gen, 21, 9).to(device).requires_grad_(True)
    kind = torch.randint(-1, 21, (15,), generator=gen).to(device)
    for cap in (None, 3.0):
        def plain(x, w):
            z = x @ w.T * 0.7
            z = cap * torch.tanh(z / cap) if cap else z
            ok = kind >= 0
            return torch.nn.functional.cross_entropy(z[ok], kind[ok], reduction="sum")
        got = torch.autograd.grad(kind_cross_entropy(x, table, kind, 0.7, cap).sum(), (x, table), create_graph=True)
        twice = torch.autograd.grad(sum(t.square().sum() for t in got), (x, table))
        wide = [t.detach().double().requires_grad_(True) for t in (x, table)]
        want = torch.autograd.grad(plain(*wide), wide, create_graph=True)
        more = torch.autograd.grad(sum(t.square().sum() for t in want), wide)
        for a, b in zip((*got, *twice), (*want, *more)):
            _within(a, b.detach(), 1e-4 * b.detach().abs().max(), "gradient")
        first = torch.autograd.grad(kind_cross_entropy(x, table, kind, 0.7, cap).sum(), (x, table))
        for i in (0, 1):
            v = _rand(gen, *(x, table)[i].shape).to(device)
            ends = [float(kind_cross_entropy(*[t.detach() + (s * 1e-2 * v if j == i else 0) for j, t in enumerate((x, table))], kind, 0.7, cap)
                          .double().sum()) for s in (1, -1)]
            along = float((first[i] * v).sum())
            assert abs((ends[0] - ends[1]) / 2e-2 - along) <= 2e-2 * (1 + abs(along))


def test_logits_are_not_kept(device):
    from equitorch_amd.nn.functional import kind_cross_entropy
    rows, kinds = 20000, 50000
    x = torch.randn(rows, 32, device=device, dtype=BF16, requires_grad=True)
    table = torch.randn(kinds, 32, device=device, dtype=BF16, requires_grad=True)
    kind = torch.randint(0, kinds, (rows,), device=device)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = kind_cross_entropy(x, table, kind)
    assert torch.cuda.max_memory_allocated() - before < rows * kinds * 2 / 20
    # a backward takes 512 MB of the logits' gradients at a time; with it two planes of 512 x 128 rows x 64 fp32 channels, as many
    # of kinds, copies of x and the results: 100 MB
    torch.autograd.grad(loss.mean(), (x, table))
    assert torch.cuda.max_memory_allocated() - before < (612 << 20) < rows * kinds * 2 / 3


def test_graph_replays(device):
    from equitorch_amd.nn.functional import kind_cross_entropy
    x = torch.randn(700, 96, device=device, dtype=BF16, requires_grad=True)
    table = torch.randn(3000, 96, device=device, dtype=BF16, requires_grad=True)
    kind = torch.randint(0, 3000, (700,), device=device)
    g = torch.rand(700, device=device)

    def step():
        loss = kind_cross_entropy(x, table, kind, 0.1)
        return (loss, *torch.autograd.grad(loss, (x, table), g))
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
            kind.copy_(torch.randint(-1000, 3000, (700,), device=device))       # another number of rows with a kind
            g.copy_(torch.rand(700, device=device))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_autocast(device):
    from equitorch_amd.nn.functional import kind_cross_entropy
    x = torch.randn(20, 16, device=device, dtype=BF16)
    table = torch.randn(9, 16, device=device, requires_grad=True)
    kind = torch.arange(20, device=device) % 9
    with torch.autocast("cuda", dtype=BF16):
        loss = kind_cross_entropy(x, table, kind)
    assert torch.equal(loss, kind_cross_entropy(x, table.to(BF16), kind))
    assert torch.autograd.grad(loss.sum(), table)[0].dtype == F32
    with pytest.raises(CgtpError):
        kind_cross_entropy(x, table, kind)


def test_refusals(device):
    from equitorch_amd.nn.functional import kind_cross_entropy
    x, w, k = torch.zeros(3, 8, device=device), torch.ones(5, 8, device=device), torch.zeros(3, dtype=torch.int64, device=device)
    for bad in ((x.double(), w.double(), k), (x, w.half(), k), (x, w, k.int()), (x, w[:, :4], k), (x, w[0], k), (x, w[:0], k), (x, w, k[:2]),
                (x, w, k[:, None]), (x[:, :0], w[:, :0], k), (x.cpu(), w, k), (x, w.cpu(), k), (x, w, k.cpu())):
        with pytest.raises(CgtpError):
            kind_cross_entropy(*bad)
    for scale, cap in ((float("nan"), None), (float("inf"), None), (1e39, None), (1.0, 0.0), (1.0, -1.0), (1.0, float("nan")), (1.0, float("inf")), (1.0, 1e-40),
                       (1e20, 1e-30)):
        with pytest.raises(CgtpError):
            kind_cross_entropy(x, w, k, scale, cap)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        kind_cross_entropy(fwd.make_dual(x, torch.ones_like(x)), w, k)


def test_layer(device):
    from equitorch_amd import nn as en
    from equitorch_amd.nn.functional import kind_cross_entropy
    table = en.Embedding(11, 8).to(device)
    m = en.KindCrossEntropy(11, 8).to(device)
    m.weight = table.weight
    x, kind = torch.randn(2, 9, 8, device=device), torch.arange(18, device=device).view(2, 9) - 3
    loss = m(x, kind)
    assert torch.equal(loss, kind_cross_entropy(x, table.weight, kind, 8 ** -0.5)) and float(loss[0, :3].detach().abs().max()) == 0
    loss.sum().backward()
    assert torch.isfinite(table.weight.grad).all()
