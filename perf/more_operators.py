"""Timed work of three operators of a training step on invariant (degree 0) node features: the root-mean-square norm that
follows a residual's addition, the softmax cross entropy over the kinds of a table, and the AdamW step over all weights.

``listed()`` gives twelve fixed cases, ``draw(rng)`` one more of the same ranges; ``prepare`` makes what a program holds
before the call, ``run`` is one pass, ``work`` the bytes and operations it cannot do without, ``exact`` the same
results in 64 bits.  With ``own`` false, ``run`` computes the operators in their plain form (elementary torch
operations in 32 bits, rounded once); with ``own`` true it calls ``equitorch_amd``.

Operators and their definitions:

* ``norm``   t = x + residual (rounded to the residual's type; t = x without one),
             out[n, c] = t[n, c] weight[c] / sqrt(mean_c t[n, c]^2 + eps).  Gradients of x, the residual and the weight from
             those of out and t.  With 8 bits, instead of out: s[n] = max_c |out[n, c]| / 448 and out[n, c] / s[n] in e4m3.
* ``loss``   z = scale x table^T, or cap tanh(scale x table^T / cap);  loss[n] = log sum_k exp z[n, k] - z[n, kind[n]], zero
             (and no gradient) for a kind outside the table.  Gradients of x and the table from one for each row.
* ``adamw``  m <- b1 m + (1 - b1) g,  v <- b2 v + (1 - b2) g^2,
             p <- p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)  over all tensors of a model.
             8 bits: m and r = sqrt(v) are kept in e4m3 with a scale, the largest magnitude / 448, for each 256 elements of a
             tensor; m rounded to nearest, r up or down at random in proportion (never from above zero to zero), the random
             bits a hash of a seed, the tensor's number, the step and the element's.  Weights in 16 bits come with copies in 32
             that the steps are taken on.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_E4M3 = torch.float8_e4m3fn
_BETAS, _DECAY, _LR, _ADAM_EPS, _NORM_EPS, _BLOCK, _SEED, _STEPS = (0.9, 0.999), 0.01, 1e-4, 1e-8, 1e-5, 256, 20011, 12


def listed():
    return [
        # Between two blocks of a small molecule at inference: a call of a few microseconds.
        {"name": "norm_molecule_forward", "op": "norm", "rows": 30, "channels": 64, "dtype": "f32", "residual": "f32",
         "pass": "forward"},
        # Training step over a large batch in mixed precision: the sum of the blocks' results stays in 32 bits.
        {"name": "norm_batch_step", "op": "norm", "rows": 65536, "channels": 256, "dtype": "bf16", "residual": "f32",
         "pass": "step"},
        # Rows of an odd length, everything in 16 bits.
        {"name": "norm_ragged_step", "op": "norm", "rows": 20011, "channels": 1001, "dtype": "f16", "residual": "f16",
         "pass": "step"},
        # Rows for a product in 8 bits at inference on a large system.
        {"name": "norm_8bit_forward", "op": "norm", "rows": 200003, "channels": 512, "dtype": "bf16", "residual": "bf16",
         "pass": "8bit"},
        # The kinds of one molecule's masked nodes, scored at inference.
        {"name": "loss_molecule_forward", "op": "loss", "rows": 30, "kinds": 100, "channels": 64, "dtype": "f32", "masked": 0.0,
         "cap": 0.0, "pass": "forward"},
        # Pretraining on elements: a batch of nodes of which most are not asked for, single precision.
        {"name": "loss_species_step", "op": "loss", "rows": 60001, "kinds": 100, "channels": 128, "dtype": "f32", "masked": 0.85,
         "cap": 0.0, "pass": "step"},
        # Pretraining on a table of local environments, mixed precision.
        {"name": "loss_environments_step", "op": "loss", "rows": 16384, "kinds": 30011, "channels": 256, "dtype": "bf16",
         "masked": 0.0, "cap": 0.0, "pass": "step"},
        # Evaluation with wide features and capped scores, odd sizes.
        {"name": "loss_evaluation_forward", "op": "loss", "rows": 5003, "kinds": 50021, "channels": 500, "dtype": "f16",
         "masked": 0.15, "cap": 30.0, "pass": "forward"},
        # A model of a few layers: dozens of small tensors, a call of a few microseconds.
        {"name": "adamw_small", "op": "adamw", "layers": 2, "kinds": 8, "channels": 64, "hidden": 128, "dtype": "f32", "bits": 32},
        # A large model in single precision.
        {"name": "adamw_large", "op": "adamw", "layers": 24, "kinds": 30011, "channels": 512, "hidden": 2048, "dtype": "f32",
         "bits": 32},
        # The same in mixed precision with states in 8 bits: 16-bit weights and gradients, 32-bit copies of the weights.
        {"name": "adamw_large_8bit", "op": "adamw", "layers": 24, "kinds": 30011, "channels": 512, "hidden": 2048, "dtype": "bf16",
         "bits": 8},
        # Tensors of odd sizes.
        {"name": "adamw_ragged_8bit", "op": "adamw", "layers": 6, "kinds": 1009, "channels": 201, "hidden": 803, "dtype": "f32",
         "bits": 8},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["norm", "loss", "loss", "adamw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        case = {"op": op, "channels": _log_int(rng, 8, 4096), "dtype": dtype, "residual": rng.choice([dtype, "f32", "none"]),
                "pass": rng.choice(["forward", "step", "step", "8bit"])}
        case["rows"] = _log_int(rng, 1, min(200003, 200003 * 128 // case["channels"]))
        return case
    if op == "adamw":
        case = {"op": op, "layers": rng.randint(1, 24), "kinds": _log_int(rng, 2, 30011), "channels": _log_int(rng, 8, 512),
                "dtype": dtype, "bits": rng.choice([32, 8])}
        case["hidden"] = rng.choice([2, 3, 4]) * case["channels"] + rng.choice([0, 0, 1, 8])
        return case
    case = {"op": op, "kinds": _log_int(rng, 2, 50021), "channels": _log_int(rng, 16, 512), "dtype": dtype,
            "masked": rng.choice([0.0, 0.0, 0.5, 0.85]), "cap": rng.choice([0.0, 0.0, 20.0]),
            "pass": rng.choice(["forward", "step", "step"])}
    # within the work of the largest listed case, a backward pass as three and 32 bits as eight times the work
    limit = 16384 * 30011 * 256 * 3 // ((8 if dtype == "f32" else 1) * (3 if case["pass"] == "step" else 1))
    most = min(limit // (case["kinds"] * case["channels"]), 500000000 // case["kinds"], 32000000 // case["channels"])
    case["rows"] = _log_int(rng, 1, max(1, min(100003, most)))
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------
def _shapes(case):
    """The tensors of a model: the kinds' table, then every layer's projections, norms and slopes."""
    c, h = case["channels"], case["hidden"]
    return [(case["kinds"], c)] + [(c, 3 * c), (c, c), (c, h), (c, h), (h, c), (c,), (c,), (max(1, c // 64),)] * case["layers"]


def _tensors(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, op, s = _DTYPES[case["dtype"]], case["op"], {"case": case}

    def randn(*shape, std=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    if op == "norm":
        n, c, step = case["rows"], case["channels"], case["pass"] == "step"
        s["x"] = randn(n, c).requires_grad_(step)
        kind = _DTYPES.get(case["residual"])
        s["residual"] = None if kind is None else randn(n, c, std=3.0, dtype=kind).requires_grad_(step)
        s["weight"] = (randn(c, std=0.2, dtype=torch.float32) + 1.0).requires_grad_(step)
        if step:
            s["ct"] = [randn(n, c), randn(n, c, dtype=dtype if kind is None else kind)]
        return s
    if op == "loss":
        n, k, c, step = case["rows"], case["kinds"], case["channels"], case["pass"] == "step"
        s["x"], s["table"] = randn(n, c).requires_grad_(step), randn(k, c).requires_grad_(step)
        # frequency of a kind ~ 1 / rank; nodes that are not asked for have kind -1
        cdf = torch.cumsum(torch.arange(1, k + 1, device=dev, dtype=torch.float64).reciprocal(), 0)
        at = torch.rand(n, generator=gen, device=dev, dtype=torch.float64) * cdf[-1]
        kind = torch.searchsorted(cdf, at).clamp_(max=k - 1)
        s["kind"] = kind.masked_fill(torch.rand(n, generator=gen, device=dev) < case["masked"], -1)
        s["scale"], s["cap"] = c ** -0.5, case["cap"] or None
        if step:
            asked = int(n * (1 - case["masked"])) or 1
            s["ct"] = torch.full((n,), 1.0 / asked, device=dev)
        return s
    # All tensors of a model lie in one buffer, each from a multiple of 256 elements on, zeros between them; gradients and
    # states lie alike.  The state is that of a dozen steps.
    shapes = _shapes(case)
    counts = [math.prod(shape) for shape in shapes]
    blocks = [-(-n // _BLOCK) for n in counts]
    first = torch.tensor([0] + blocks).cumsum(0)
    real = torch.zeros(int(first[-1]) * _BLOCK, dtype=torch.bool)
    for at, n in zip((first[:-1] * _BLOCK).tolist(), counts):
        real[at:at + n] = True
    real = real.to(dev)
    total = real.numel()
    s["places"] = list(zip((first[:-1] * _BLOCK).tolist(), counts, shapes))
    # the number of a block's tensor, and of its first element in it
    per_block = torch.repeat_interleave(torch.arange(len(shapes)), torch.tensor(blocks))
    s["tensor"] = per_block.to(dev)
    s["element"] = ((torch.arange(len(per_block)) - first[per_block]) * _BLOCK).to(dev)
    weight = randn(total, std=0.05, dtype=torch.float32) * real
    s["p"] = weight.to(dtype)
    s["master"] = None if dtype == torch.float32 else weight
    size = 1e-3 * torch.exp(randn(total // _BLOCK, 1, dtype=torch.float32)).expand(-1, _BLOCK).reshape(-1)   # of a block's gradients
    s["g"] = (randn(total, dtype=torch.float32) * size * real).to(dtype)
    m = randn(total, std=0.3, dtype=torch.float32) * size * real
    v = (randn(total, std=0.2, dtype=torch.float32) + 1.0).square() * size.square() * real * (1 - _BETAS[1] ** _STEPS)
    s["step"] = torch.full((len(shapes),), float(_STEPS), device=dev)
    if case["bits"] == 32:
        s["exp_avg"], s["exp_avg_sq"] = m, v
    else:
        for name, value in (("exp_avg", m), ("root_avg_sq", v.sqrt())):
            scale, inverse = _block_scales(value.view(-1, _BLOCK))
            s[name] = (value.view(-1, _BLOCK) * inverse[:, None]).clamp(-448, 448).to(_E4M3).view(-1)
            s[name + "_scale"] = scale
    return s


def prepare(case, seed):
    s = _tensors(case, seed)
    if own and case["op"] == "adamw":
        from equitorch_amd.optim import AdamW
        params = [torch.nn.Parameter(s["p"][at:at + n].view(shape)) for at, n, shape in s["places"]]
        s["optimizer"] = opt = AdamW(params, lr=_LR, betas=_BETAS, eps=_ADAM_EPS, weight_decay=_DECAY, state_bits=case["bits"],
                                     master=s["master"] is not None, seed=_SEED)
        wide = ["exp_avg", "exp_avg_sq"] if case["bits"] == 32 else ["exp_avg", "root_avg_sq"]
        wide += ["master"] if s["master"] is not None else []
        for i, (p, (at, n, shape)) in enumerate(zip(params, s["places"])):
            p.grad = s["g"][at:at + n].view(shape)
            opt.state[p] = {"step": s["step"][i], **{name: s[name][at:at + n].view(shape) for name in wide}}
            if case["bits"] == 8:
                a, b = at // _BLOCK, at // _BLOCK + -(-n // _BLOCK)
                opt.state[p].update({name + "_scale": s[name + "_scale"][a:b] for name in wide[:2]})
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------
def _block_scales(rows):
    """The scale of each row of values, its largest magnitude / 448 (zero for zeros, not below the normal numbers), and its inverse."""
    top = rows.abs().amax(-1)
    scale = torch.where(top > 0, (top / 448.0).clamp(min=2.0 ** -126), torch.zeros_like(top))
    return scale, torch.where(top > 0, 1.0 / scale.masked_fill(top == 0, 1.0), torch.zeros_like(top))


def _plain_norm(x, residual, weight, kind):
    t = x if residual is None else x + residual
    t = t + (t.detach().to(kind).float() - t.detach())          # rounded to its type, gradients as they are
    return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + _NORM_EPS) * weight, t


def _plain_loss(s, x, table):
    z = x @ table.T * s["scale"]
    if s["cap"]:
        z = s["cap"] * torch.tanh(z / s["cap"])
    top = z.detach().amax(-1, keepdim=True)
    lse = torch.exp(z - top).sum(-1).log() + top[:, 0]
    asked = s["kind"] >= 0
    at = z.gather(1, s["kind"].clamp(min=0)[:, None])[:, 0]
    return torch.where(asked, lse - at, torch.zeros_like(lse))


def _random_bits(seed, tensor, step, element):
    """20 random bits of each element, by 32-bit arithmetic held in 64."""
    def mix(h):
        h = (h ^ (h >> 16)) * 0x9C8F2D35 & 0xFFFFFFFF
        h = (h ^ (h >> 15)) * 0xB5297A4D & 0xFFFFFFFF
        return h ^ (h >> 16)
    key = mix((seed * 0x85157AF5 + tensor * 0x9E3779B1 + step * 0xC2B2AE63) & 0xFFFFFFFF)
    return mix((key + element * 0x9E3779B1) & 0xFFFFFFFF) >> 12


def _round_at_random(value, bits):
    """Values in 0 .. 448 to e4m3, up or down in proportion; above zero not to zero."""
    normal = ((value.view(torch.int32) + bits) & -(1 << 20)).view(torch.float32)
    small = torch.floor(value * 512.0 + bits.float() * 2.0 ** -20) / 512.0
    q = torch.where(value < 2.0 ** -6, small.clamp(min=2.0 ** -9), normal)
    return torch.where(value > 0, q, torch.zeros_like(q)).clamp(max=448.0).to(_E4M3)


def _plain_adamw(s):
    case, (b1, b2) = s["case"], _BETAS
    s["step"] += 1
    g, step = s["g"].float(), s["step"].double()
    if case["bits"] == 32:
        m, v = s["exp_avg"], s["exp_avg_sq"]
    else:
        m = s["exp_avg"].float().view(-1, _BLOCK) * s["exp_avg_scale"][:, None]
        v = (s["root_avg_sq"].float().view(-1, _BLOCK) * s["root_avg_sq_scale"][:, None]).square()
        g = g.view(-1, _BLOCK)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    of_block = lambda t: t.float()[s["tensor"]][:, None]                                              # noqa: E731
    size, root = of_block(_LR / (1 - b1 ** step)), of_block((1 - b2 ** step).rsqrt())
    p = s["p"].float() if s["master"] is None else s["master"]
    r = v.sqrt()
    update = m.view(-1, _BLOCK) / (r.view(-1, _BLOCK) * root + _ADAM_EPS)
    p.copy_((p.view(-1, _BLOCK) * (1 - _LR * _DECAY) - size * update).view(-1))
    if p is not s["p"]:
        s["p"].copy_(p)
    if case["bits"] == 32:
        s["exp_avg"].copy_(m)
        s["exp_avg_sq"].copy_(v)
        return
    scale, inverse = _block_scales(m)
    s["exp_avg_scale"].copy_(scale)
    s["exp_avg"].copy_((m * inverse[:, None]).clamp(-448, 448).to(_E4M3).view(-1))
    scale, inverse = _block_scales(r)
    s["root_avg_sq_scale"].copy_(scale)
    element = s["element"][:, None] + torch.arange(_BLOCK, device=g.device)
    bits = _random_bits(_SEED, s["tensor"][:, None], s["step"].long()[s["tensor"]][:, None], element).int()
    s["root_avg_sq"].copy_(_round_at_random((r * inverse[:, None]).clamp(max=448.0), bits).view(-1))


def _state(s):
    names = ["p", "master", "step", "exp_avg", "exp_avg_sq", "exp_avg_scale", "root_avg_sq", "root_avg_sq_scale"]
    return {n: s[n] for n in names if s.get(n) is not None}


def run(s):
    case = s["case"]
    if case["op"] == "adamw":
        with torch.no_grad():
            if own:
                s["optimizer"].step()
            else:
                _plain_adamw(s)
        return _state(s)
    if case["op"] == "norm":
        given = [s["x"], s["residual"], s["weight"]]
        kind = (s["x"] if s["residual"] is None else s["residual"]).dtype
    else:
        given = [s["x"], s["table"]]
    present = [t for t in given if t is not None]
    if own:
        from equitorch_amd.nn import functional as F
        if case["pass"] == "8bit":
            with torch.no_grad():
                return F.add_rms_norm_8bit(*given, eps=_NORM_EPS)
        with torch.set_grad_enabled(case["pass"] == "step"):
            outs = F.add_rms_norm(*given, eps=_NORM_EPS) if case["op"] == "norm" else \
                [F.kind_cross_entropy(s["x"], s["table"], s["kind"], s["scale"], s["cap"])]
        if case["pass"] == "forward":
            return outs
        return (*outs, *torch.autograd.grad(outs, present, s["ct"]))
    step = case["pass"] == "step"
    wide = [None if t is None else t.detach().float().requires_grad_(step) for t in given]
    with torch.set_grad_enabled(step):
        outs = _plain_norm(*wide, kind) if case["op"] == "norm" else [_plain_loss(s, *wide)]
    if case["pass"] == "8bit":
        scale, inverse = _block_scales(outs[0])
        return (outs[0] * inverse[:, None]).clamp(-448, 448).to(_E4M3), scale, outs[1].to(kind)
    types = [s["x"].dtype, kind] if case["op"] == "norm" else [torch.float32]
    rounded = [o.detach().to(t) for o, t in zip(outs, types)]
    if not step:
        return rounded
    ct = [t.float() for t in s["ct"]] if case["op"] == "norm" else s["ct"]
    grads = torch.autograd.grad(outs, [t for t in wide if t is not None], ct)
    return (*rounded, *[g.to(t.dtype) for g, t in zip(grads, present)])


# ---- what a pass cannot do without ----------------------------------------------------------------------------
def work(case):
    b = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        n, c = case["rows"], case["channels"]
        r = {"none": 0, "f32": 4}.get(case["residual"], 2)
        row = b + r + (1 if case["pass"] == "8bit" else b) + r             # x, the residual; out, t
        if case["pass"] == "step":      # the gradients of out and t in; those of x and, where its type is another, the residual out
            row += b + (r or b) + b + (r if r != b else 0)
        return {"bytes": n * c * row + 4 * c, "flops": n * c * (16 if case["pass"] == "step" else 5)}
    if case["op"] == "loss":
        n, k, c = max(1, round(case["rows"] * (1 - case["masked"]))), case["kinds"], case["channels"]
        step = case["pass"] == "step"
        once = (n + k) * c * b
        return {"bytes": (2 if step else 1) * once + 12 * case["rows"], "flops": (6.0 if step else 2.0) * n * k * c}
    n = sum(math.prod(shape) for shape in _shapes(case))
    each = b + (8 if b == 4 else 8 + b) + (16 if case["bits"] == 32 else 4 + 16 / _BLOCK)      # gradient, weights, states
    return {"bytes": n * each, "flops": 15.0 * n}


# ---- 64-bit results -------------------------------------------------------------------------------------------
def _e4m3(x):
    """The nearest values of e4m3 to those of x, by their binary exponents (ties to even)."""
    _, e = torch.frexp(x)
    unit = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return (torch.round(x / unit) * unit).clamp(-448, 448)


def _by_448(rows):
    top = rows.abs().amax(-1)
    scale = torch.where(top > 0, (top / 448).clamp(min=2.0 ** -126), 0.0 * top)
    return scale, rows / torch.where(top > 0, scale, 1.0 + 0.0 * top)[:, None]


def _exact_norm(s):
    case, w = s["case"], s["weight"].detach().double()
    x = s["x"].detach()
    # the sum is exact in 64 bits: t is its rounding, and what follows is a function of t
    t = x if s["residual"] is None else (x.double() + s["residual"].detach().double()).to(s["residual"].dtype)
    t = t.double()
    inv = 1 / (t.pow(2).sum(1, keepdim=True) / case["channels"] + _NORM_EPS).sqrt()
    out = t * inv * w
    if case["pass"] == "8bit":
        scale, rows = _by_448(out)
        return _e4m3(rows), scale, t
    if case["pass"] == "forward":
        return out, t
    g, gt = (c.double() for c in s["ct"])
    u = g * w
    gx = gt + inv * (u - t * inv.pow(2) * (u * t).sum(1, keepdim=True) / case["channels"])
    gw = (g * t * inv).sum(0)
    return (out, t, gx, gw) if s["residual"] is None else (out, t, gx, gx, gw)


def _exact_loss(s):
    case = s["case"]
    x, w, kind, cap = s["x"].detach().double(), s["table"].detach().double(), s["kind"], s["cap"]
    loss = torch.zeros(case["rows"], dtype=torch.float64, device=x.device)
    gx, gw = torch.zeros_like(x), torch.zeros_like(w)
    asked = torch.nonzero(kind >= 0)[:, 0]
    for rows in asked.split(max(1, 2 ** 27 // case["kinds"])):
        z = (x[rows] @ w.T) * s["scale"]
        th = torch.tanh(z / cap) if cap else None
        z = cap * th if cap else z
        logp = torch.log_softmax(z, 1)
        at = torch.arange(len(rows), device=x.device)
        loss[rows] = -logp[at, kind[rows]]
        if case["pass"] == "step":
            gz = logp.exp()
            gz[at, kind[rows]] -= 1
            gz *= s["ct"][rows].double()[:, None] * s["scale"]
            if cap:
                gz *= 1 - th * th
            gx[rows] = gz @ w
            gw += gz.T @ x[rows]
    return (loss, gx, gw) if case["pass"] == "step" else [loss]


def _exact_adamw(s):
    case, (b1, b2), n = s["case"], _BETAS, _STEPS + 1
    rows = lambda t: t.double().view(-1, _BLOCK)                                                       # noqa: E731
    g, p = rows(s["g"]), rows(s["p"] if s["master"] is None else s["master"])
    if case["bits"] == 32:
        m, v = rows(s["exp_avg"]), rows(s["exp_avg_sq"])
    else:
        m = rows(s["exp_avg"].float()) * s["exp_avg_scale"].double()[:, None]
        v = (rows(s["root_avg_sq"].float()) * s["root_avg_sq_scale"].double()[:, None]) ** 2
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    p = p - _LR * _DECAY * p - _LR / (1 - b1 ** n) * m / (torch.sqrt(v / (1 - b2 ** n)) + _ADAM_EPS)
    got = {"p": p.view(-1), "step": torch.full_like(s["step"], n, dtype=torch.float64)}
    if s["master"] is not None:
        got["master"] = p.view(-1)
    if case["bits"] == 32:
        return {**got, "exp_avg": m.view(-1), "exp_avg_sq": v.view(-1)}
    scale, q = _by_448(m)
    got.update(exp_avg=_e4m3(q).view(-1), exp_avg_scale=scale)
    scale, q = _by_448(v.sqrt())
    element = s["element"][:, None] + torch.arange(_BLOCK, device=g.device)
    part = _random_bits(_SEED, s["tensor"][:, None], n, element).double() / 2 ** 20
    # what lies below a value by less than the random part of a unit of its binary exponent goes up
    _, e = torch.frexp(q)
    unit = torch.ldexp(torch.ones_like(q), (e - 4).clamp(min=-9))
    r = (torch.floor(q / unit + part) * unit).clamp(max=448)
    r = torch.where(q > 0, r.clamp(min=2.0 ** -9), torch.zeros_like(r))
    got.update(root_avg_sq=r.view(-1), root_avg_sq_scale=scale)
    return got


def exact(case, seed):
    s = _tensors(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "loss": _exact_loss, "adamw": _exact_adamw}[case["op"]](s)
