"""States in 8 bits of gradients whose sizes in a block differ widely: bit for bit the formulas in elementary operations of 32 bits."""
import pytest
import torch

from equitorch_amd.optim import AdamW

pytestmark = pytest.mark.gpu


def _mixed(h):
    h = (h ^ (h >> 16)) * 0x9C8F2D35 & 0xFFFFFFFF
    h = (h ^ (h >> 15)) * 0xB5297A4D & 0xFFFFFFFF
    return h ^ (h >> 16)


def _scales(x):
    most = x.abs().amax(1)
    scale = (most * (1 / 448)).clamp(min=2.0 ** -126)
    return scale, (1.0 / scale)[:, None]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_roots_below_the_normal_numbers_of_e4m3(device, dtype):
    """Below 2^-6 of the unit the values are multiples of 2^-9: the random bits are added with 2^-6 on top, which is then taken off."""
    rows, seed, (b1, b2) = 300, 5, (0.9, 0.95)
    n = rows * 256
    gen = torch.Generator().manual_seed(11)
    p = torch.nn.Parameter(torch.randn(n, generator=gen).to(device, dtype))
    opt = AdamW([p], lr=1e-3, betas=(b1, b2), state_bits=8, seed=seed)
    m = v = torch.zeros(rows, 256, device=device)
    element = torch.arange(n, device=device).view(rows, 256)
    for step in range(1, 6):
        g = (torch.randn(n, generator=gen) * 2.0 ** (-20 * torch.rand(n, generator=gen))).to(device, dtype)
        p.grad = g
        opt.step()
        g = g.float().view(rows, 256)
        m, v = m * b1 + g * (1 - b1), v * b2 + g * g * (1 - b2)
        state = opt.state[p]
        scale, inverse = _scales(m)
        codes = (m * inverse).clamp(-448, 448).to(torch.float8_e4m3fn)
        assert torch.equal(state["exp_avg_scale"], scale) and torch.equal(state["exp_avg"].view(rows, 256).view(torch.uint8), codes.view(torch.uint8))
        m = codes.float() * scale[:, None]
        scale, inverse = _scales(v.sqrt())
        q = (v.sqrt() * inverse).clamp(max=448.0)
        key = _mixed(torch.tensor(seed * 0x85157AF5 + step * 0xC2B2AE63, device=device) & 0xFFFFFFFF)
        bits = (_mixed((key + element * 0x9E3779B1) & 0xFFFFFFFF) >> 12).int()
        lift = (q < 2.0 ** -6).float() * 2.0 ** -6
        want = (((q + lift).view(torch.int32) + bits) & -(1 << 20)).view(torch.float32) - lift
        want = torch.where(q > 0, want.clamp(min=2.0 ** -9), 0.0)
        got = state["root_avg_sq"].view(rows, 256).float()
        assert torch.equal(state["root_avg_sq_scale"], scale) and torch.equal(got, want)
        assert step > 1 or (q < 2.0 ** -6).float().mean() > 0.1
        v = (got * scale[:, None]).square()
