"""Cross entropy over kinds with caps far above the logits, against its definition in 64 bits.

A logit's error may grow with the logit, not with the cap: tolerances are the roundings of 2^-24 of what enters a logit, and those of the
operands' type where `softmax - one` and the rows times their gradient enter a product."""
import pytest
import torch

from helpers import stable_seed

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
EPS = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
U = 2.0 ** -24
WALK_CAP = 256.0      # up to it kernels whose tangent errs some roundings of 1


def _within(got, want, bound, what):
    got = got.detach().cpu().double()
    excess = float(((got - want).abs() - bound).max())
    assert excess <= 0 and torch.isfinite(got).all(), f"{what}: {excess:.3e} over the bound"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("channels", [24, 200, 300, 512, 600])
@pytest.mark.parametrize("cap", [255.0, 256.0, 257.0, 1e4, 1e6, 1e9])
def test_caps_far_above_the_logits(device, dtype, channels, cap):
    from equitorch_amd.nn.functional import kind_cross_entropy
    gen = torch.Generator().manual_seed(stable_seed(channels, int(cap)))
    n, k, scale = 70, 301, -2.0 * channels ** -0.5
    x, w = (torch.randn(s, channels, generator=gen, dtype=F64).to(dtype) for s in (n, k))
    kind = torch.randint(0, k, (n,), generator=gen)
    g = torch.rand(n, generator=gen) + 0.5
    leaves = [t.to(device).requires_grad_(True) for t in (x, w)]
    loss = kind_cross_entropy(*leaves, kind.to(device), scale, cap)
    grads = torch.autograd.grad(loss, leaves, g.to(device))

    x, w, g = x.double(), w.double(), g.double()[:, None]
    raw = x @ w.T * scale
    th = torch.tanh(raw / cap)
    z = cap * th
    # a product over the channels, scale and tangent (ten roundings of itself), to the base 2 and less the maximum
    err = (channels + 4) * U * (x.abs() @ w.abs().T) * abs(scale) + 10 * U * z.abs() + 4 * U * z.abs().amax(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    delta = err.amax(1, keepdim=True) + (k / 4 + 40) * U                 # of lse: its terms' errors, and a sum in chains of k / 4
    want = (lse - z.gather(1, kind[:, None]))[:, 0]
    _within(loss, want, (delta + err.gather(1, kind[:, None]) + 4 * U * (lse.abs() + want.abs()[:, None]))[:, 0], "loss")
    if cap <= WALK_CAP:
        err = err + 12 * U * cap
    one = torch.zeros_like(z).scatter_(1, kind[:, None], 1.0)
    p, slope = (z - lse).exp(), 1 - th * th
    dz = (p - one) * slope
    off = 2 * p * (err + delta + 2 * U * (z - lse).abs()) + 2 * U * one + 24 * U * (p + one)      # 24: the slope's
    off = off + EPS[dtype] * (dz.abs() + off) + (2.0 ** -40 if dtype == F16 else 2.0 ** -120)
    least = 2.0 ** -25 if dtype == F16 else 0.0
    want = g * scale * (dz @ w)
    size = g * abs(scale) * ((off + (k + 4) * U * dz.abs()) @ w.abs())
    _within(grads[0], want, EPS[dtype] * (want.abs() + size) + size + least, "grad_x")
    xg = g * x
    rounding = EPS[dtype] * xg.abs() + float(g.max()) * least
    want = scale * (dz.T @ xg)
    size = abs(scale) * ((off + (n + 8) * U * dz.abs()).T @ (xg.abs() + rounding) + dz.abs().T @ rounding)
    _within(grads[1], want, EPS[dtype] * (want.abs() + size) + size + least, "grad_table")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_logit_near_the_cap_leaves_the_others_theirs(device, dtype):
    """A kind whose logit is far below the others, near the cap: the others' logits keep their bits, and the loss theirs."""
    from equitorch_amd.nn.functional import kind_cross_entropy
    gen = torch.Generator().manual_seed(5)
    n, k, c, cap = 40, 100, 32, 4096.0
    x, w = (torch.randn(s, c, generator=gen, dtype=F64).to(dtype) for s in (n, k))
    x[:, 0], w[:, 0] = 64.0, 0.0
    w[17, 0] = -64.0                                                     # a logit of some -4096
    kind = torch.randint(18, k, (n,), generator=gen)
    leaves = [t.to(device).requires_grad_(True) for t in (x, w)]
    loss = kind_cross_entropy(*leaves, kind.to(device), 1.0, cap)
    (gx,) = torch.autograd.grad(loss, leaves[:1], torch.ones(n, device=device))
    x, w = x.double(), w.double()
    others = torch.arange(k) != 17
    raw = (x @ w.T)[:, others]
    z = cap * torch.tanh(raw / cap)
    err = (c + 4) * U * (x.abs() @ w.abs().T)[:, others] + 14 * U * z.abs().amax(1, keepdim=True)
    at = (kind - 1)[:, None]
    lse = torch.logsumexp(z, 1, keepdim=True)                            # the kind far below adds exp(-3000)
    delta = err.amax(1, keepdim=True) + (k / 4 + 40) * U
    want = (lse - z.gather(1, at))[:, 0]
    _within(loss, want, (delta + err.gather(1, at) + 4 * U * (lse.abs() + want.abs()[:, None]))[:, 0], "loss")
    one = torch.zeros_like(z).scatter_(1, at, 1.0)
    p, slope = (z - lse).exp(), 1 - (z / cap).square()
    dz = (p - one) * slope
    off = 2 * p * (err + delta + 2 * U * (z - lse).abs()) + 2 * U * one + 24 * U * (p + one)
    off = off + EPS[dtype] * (dz.abs() + off) + (2.0 ** -40 if dtype == F16 else 2.0 ** -120)
    want = dz @ w[others]
    size = (off + (k + 4) * U * dz.abs()) @ w[others].abs()
    _within(gx, want, EPS[dtype] * (want.abs() + size) + size + (2.0 ** -25 if dtype == F16 else 0.0), "grad_x")
