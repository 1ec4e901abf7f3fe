"""Timed work of the operators on invariant (degree 0) node features: embedding of node kinds, attention among the
nodes of a structure, and the gated feed-forward block.

``listed()`` gives twelve fixed cases, ``draw(rng)`` one more of the same ranges; ``prepare`` makes what a program holds
before the call, ``run`` is one pass, ``work`` the bytes and operations it cannot do without, ``exact`` the same
results in 64 bits.  With ``own`` false, ``run`` computes the operators in their plain form (elementary torch
operations in 32 bits, rounded once); with ``own`` true it calls ``equitorch_amd.nn.functional``.

Operators and their definitions:

* ``embed``   out[i] = scale * table[kind[i]];  grad_table[t] = scale * sum of grad_out[i] over the i of kind t.
* ``attn``    nodes of many structures one after the other; every query of a structure sees all of its keys.
              s_ij = cap * tanh(a q_i.k_j / cap) - slope_h |r_i - r_j|,  a = D^-1/2,  out_i = sum_j softmax_j(s_ij) v_j,
              zero for a structure without keys.  Several query heads may share one head of keys and values.  Gradients
              of q, k, v, the positions and the slopes.
* ``ff``      y = (silu(x Wg) * (x Wu)) Wd;  gradients of x and of the three weights.
"""
import math
import random

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # The kinds of one small molecule's atoms at inference: a call of a few microseconds.
        {"name": "embed_molecule_forward", "op": "embed", "rows": 30, "kinds": 100, "channels": 64, "dtype": "f32",
         "skew": 1.0, "pass": "forward"},
        # Training step over a batch of structures: few kinds, most rows in a handful of them.
        {"name": "embed_species_step", "op": "embed", "rows": 60001, "kinds": 100, "channels": 128, "dtype": "f32",
         "skew": 2.0, "pass": "step"},
        # A table of local environments instead of elements, mixed precision: many kinds, most of them rare.
        {"name": "embed_environments_step", "op": "embed", "rows": 1000003, "kinds": 30011, "channels": 256,
         "dtype": "bf16", "skew": 1.1, "pass": "step"},
        # Readout of a batch of molecules: one query for each structure, some structures empty.
        {"name": "attn_readout_forward", "op": "attn", "structures": 64, "shortest": 0, "longest": 400,
         "queries": "one", "heads": 8, "kv_heads": 8, "dim": 32, "dtype": "f32", "bias": True, "cap": 0.0,
         "pass": "forward"},
        # One query over all the nodes of one large system, keys and values shared by four heads each.
        {"name": "attn_one_query_forward", "op": "attn", "structures": 1, "shortest": 200003, "longest": 200003,
         "queries": "one", "heads": 8, "kv_heads": 2, "dim": 64, "dtype": "bf16", "bias": True, "cap": 30.0,
         "pass": "forward"},
        # Training step on small molecules: hundreds of short sequences of odd lengths, narrow heads, forces.
        {"name": "attn_molecules_step", "op": "attn", "structures": 1024, "shortest": 5, "longest": 29,
         "queries": "all", "heads": 8, "kv_heads": 8, "dim": 16, "dtype": "f32", "bias": True, "cap": 0.0,
         "pass": "step"},
        # The same on drug-sized molecules in mixed precision, with capped scores.
        {"name": "attn_ligands_step", "op": "attn", "structures": 300, "shortest": 40, "longest": 250,
         "queries": "all", "heads": 8, "kv_heads": 8, "dim": 32, "dtype": "bf16", "bias": True, "cap": 30.0,
         "pass": "step"},
        # A few bulk structures of thousands of atoms.
        {"name": "attn_bulk_step", "op": "attn", "structures": 3, "shortest": 2000, "longest": 5000,
         "queries": "all", "heads": 8, "kv_heads": 4, "dim": 64, "dtype": "bf16", "bias": True, "cap": 30.0,
         "pass": "step"},
        # Inference on one large system, wide heads, no bias and no cap.
        {"name": "attn_system_forward", "op": "attn", "structures": 1, "shortest": 12007, "longest": 12007,
         "queries": "all", "heads": 16, "kv_heads": 4, "dim": 128, "dtype": "f16", "bias": False, "cap": 0.0,
         "pass": "forward"},
        # The readout network on a single row.
        {"name": "ff_row_forward", "op": "ff", "rows": 1, "channels": 256, "hidden": 1024, "dtype": "bf16",
         "pass": "forward"},
        # Training step over the nodes of a batch in single precision, ragged row count.
        {"name": "ff_nodes_step", "op": "ff", "rows": 3001, "channels": 128, "hidden": 512, "dtype": "f32",
         "pass": "step"},
        # A large batch in mixed precision.
        {"name": "ff_batch_step", "op": "ff", "rows": 65536, "channels": 256, "hidden": 1024, "dtype": "bf16",
         "pass": "step"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["embed", "attn", "attn", "ff", "ff"])
    case = {"op": op, "dtype": rng.choice(["f32", "bf16", "f16"]), "pass": rng.choice(["step", "step", "forward"])}
    if op == "embed":
        case.update(kinds=_log_int(rng, 2, 50000), channels=_log_int(rng, 8, 512), skew=rng.choice([0.0, 1.0, 1.5]))
        case["rows"] = _log_int(rng, 1, min(1000003, 256000000 // case["channels"]))
        return case
    if op == "ff":
        case.update(channels=_log_int(rng, 16, 512), hidden=_log_int(rng, 32, 2048))
        limit = 65536 * 256 * 1024 // (8 if case["dtype"] == "f32" else 1)
        case["rows"] = _log_int(rng, 1, min(65536, limit // (case["channels"] * case["hidden"])))
        return case
    groups = rng.choice([1, 1, 2, 4])
    case.update(kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([8, 16, 24, 32, 48, 64, 64, 80, 96, 128]),
                bias=rng.random() < 0.7, cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                queries=rng.choice(["all", "all", "all", "one"]))
    case["heads"] = case["kv_heads"] * groups
    # length first, within the work of the largest listed case (a backward pass as four, 32 bits as four times the
    # work), then as many structures as that leaves room for
    work_of_pair = case["heads"] * (case["dim"] + 32) * (4 if case["pass"] == "step" else 1) \
        * (4 if case["dtype"] == "f32" else 1)
    pairs = 3.6e11 / work_of_pair
    one = case["queries"] == "one"
    longest = _log_int(rng, 1, 100000 if one else min(6000, int(pairs ** 0.5)))
    case["longest"], case["shortest"] = longest, rng.choice([0, longest // 4, longest])
    most = min(2000, 200000 // longest, int(pairs / (longest if one else longest * longest)))
    case["structures"] = _log_int(rng, 1, max(1, most))
    return case


# ---- sizes ----------------------------------------------------------------------------------------------------
def _lengths(case):
    """Keys of every structure, fixed by the case alone; the first has the greatest length."""
    rng = random.Random(case["structures"] * 1000003 + case["longest"])
    return [case["longest"]] + [rng.randint(case["shortest"], case["longest"]) for _ in range(case["structures"] - 1)]


def _sizes(case):
    keys = _lengths(case)
    return (keys if case["queries"] == "all" else [1] * len(keys)), keys


def _pointer(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


# ---- inputs ---------------------------------------------------------------------------------------------------
def prepare(case, seed):
    s = _tensors(case, seed)
    if case["op"] == "attn":
        len_q, len_k = _sizes(case)
        ptr_q, ptr_k, dev = _pointer(len_q), _pointer(len_k), s["qkv"][0].device
        if own:
            from equitorch_amd.nn.functional import AttentionPlan
            ptr = torch.tensor(ptr_k, device=dev)
            alone = case["queries"] == "all"
            s["plan"] = AttentionPlan(ptr) if alone else AttentionPlan(torch.tensor(ptr_q, device=dev), ptr)
        else:
            s["buckets"], s["inverse"] = _buckets(len_q, len_k, ptr_q, ptr_k, case["heads"], dev)
    return s


def _tensors(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, op, step = _DTYPES[case["dtype"]], case["op"], case["pass"] == "step"
    s = {"case": case}

    def randn(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    if op == "embed":
        # frequency of a kind ~ rank^-skew, the ranks in an order of their own
        weights = torch.arange(1, case["kinds"] + 1, device=dev, dtype=torch.float64) ** -case["skew"]
        cdf = torch.cumsum(weights, 0) / weights.sum()
        u = torch.rand(case["rows"], generator=gen, device=dev, dtype=torch.float64)
        rank = torch.searchsorted(cdf, u).clamp_(max=case["kinds"] - 1)
        s["kind"] = torch.randperm(case["kinds"], generator=gen, device=dev)[rank]
        s["table"] = randn(case["kinds"], case["channels"]).requires_grad_(step)
        s["scale"] = case["channels"] ** 0.5
        if step:
            s["ct"] = randn(case["rows"], case["channels"])
        return s
    if op == "ff":
        c, h = case["channels"], case["hidden"]
        s["x"] = randn(case["rows"], c).requires_grad_(step)
        s["w"] = [randn(c, h, std=c ** -0.5), randn(c, h, std=c ** -0.5), randn(h, c, std=h ** -0.5)]
        if step:
            for t in s["w"]:
                t.requires_grad_(True)
            s["ct"] = randn(case["rows"], c)
        return s
    len_q, len_k = _sizes(case)
    nq, nk, hq, hk, d = sum(len_q), sum(len_k), case["heads"], case["kv_heads"], case["dim"]
    # queries, keys and values as one projection of the features leaves them: slices of one tensor
    if case["queries"] == "all":
        q, k, v = randn(nk, hq + 2 * hk, d).split([hq, hk, hk], dim=1)
    else:
        q = randn(nq, hq, d)
        k, v = randn(nk, 2 * hk, d).split([hk, hk], dim=1)
    s["qkv"] = [t.detach().requires_grad_(step) for t in (q, k, v)]
    s["pos"], s["pos_k"], s["slope"] = None, None, None
    if case["bias"]:
        # atoms uniform in a cube of 8 cubic units an atom; a query of its own sits near the middle
        side = torch.tensor(len_k, device=dev, dtype=torch.float32).clamp_(min=1).pow(1 / 3) * 2.0
        per_key = torch.repeat_interleave(side, torch.tensor(len_k, device=dev), output_size=nk)
        pos_k = (torch.rand(nk, 3, generator=gen, device=dev) - 0.5) * per_key[:, None]
        pos = pos_k if case["queries"] == "all" else torch.rand(nq, 3, generator=gen, device=dev) - 0.5
        s["pos"] = pos.requires_grad_(step)
        s["pos_k"] = None if case["queries"] == "all" else pos_k.requires_grad_(step)
        s["slope"] = torch.rand(hq, generator=gen, device=dev).mul_(0.5).requires_grad_(step)
    s["scale"], s["cap"] = d ** -0.5, case["cap"] or None
    if step:
        s["ct"] = randn(nq, hq, d)
    return s


def _buckets(len_q, len_k, ptr_q, ptr_k, heads, dev):
    """Structures of similar length together, padded to the longest of the bucket: index and mask tensors."""
    groups = {}
    for i, (a, b) in enumerate(zip(len_q, len_k)):
        if a:
            groups.setdefault((a - 1).bit_length() * 64 + max(b - 1, 0).bit_length(), []).append(i)
    buckets, order = [], []
    for members in groups.values():
        lq, lk = max(len_q[i] for i in members), max(1, max(len_k[i] for i in members))
        most = max(1, 2 ** 28 // (heads * lq * lk))
        for at in range(0, len(members), most):
            part = members[at:at + most]
            n_q = torch.tensor([len_q[i] for i in part])[:, None]
            n_k = torch.tensor([len_k[i] for i in part])[:, None]
            col_q, col_k = torch.arange(lq)[None], torch.arange(lk)[None]
            row_q = torch.tensor([ptr_q[i] for i in part])[:, None] + col_q
            row_k = torch.tensor([ptr_k[i] for i in part])[:, None] + col_k
            row_k = torch.where(col_k < n_k, row_k, torch.zeros_like(row_k))
            real = (col_q < n_q).flatten()
            order.append(row_q.flatten()[real])
            row_q = torch.where(col_q < n_q, row_q, torch.zeros_like(row_q))
            buckets.append({"rows_q": row_q.to(dev), "rows_k": row_k.to(dev), "keep": (col_k < n_k).to(dev),
                            "real": real.nonzero().flatten().to(dev)})
    order = torch.cat(order) if order else torch.zeros(0, dtype=torch.int64)
    return buckets, torch.argsort(order).to(dev)


# ---- plain forms ----------------------------------------------------------------------------------------------
def _plain_attention(s, q, k, v, pos, pos_k, slope):
    outs, group = [], q.shape[1] // k.shape[1]
    pos_k = pos if pos_k is None else pos_k
    for b in s["buckets"]:
        qb = q[b["rows_q"]].transpose(1, 2)                                                        # B, H, Lq, D
        kb = k[b["rows_k"]].transpose(1, 2).repeat_interleave(group, dim=1)
        vb = v[b["rows_k"]].transpose(1, 2).repeat_interleave(group, dim=1)
        score = torch.matmul(qb, kb.transpose(2, 3)) * s["scale"]
        if s["cap"]:
            score = s["cap"] * torch.tanh(score / s["cap"])
        if slope is not None:
            diff = pos[b["rows_q"]][:, :, None] - pos_k[b["rows_k"]][:, None]
            d2 = (diff * diff).sum(-1)
            dist = torch.where(d2 > 0, d2, torch.ones_like(d2)).sqrt() * (d2 > 0)
            score = score - slope[:, None, None] * dist[:, None]
        score = score.masked_fill(~b["keep"][:, None, None], -math.inf)
        top = score.amax(-1, keepdim=True).detach()
        p = torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top)))
        total = p.sum(-1, keepdim=True)
        out = torch.matmul(p, vb) / torch.where(total > 0, total, torch.ones_like(total))
        outs.append(out.transpose(1, 2).reshape(-1, *q.shape[1:])[b["real"]])
    return torch.cat(outs)[s["inverse"]]


def _plain(s, op, inputs):
    """The operator on 32-bit copies of its differentiable inputs."""
    if op == "embed":
        return inputs[0][s["kind"]] * s["scale"]
    if op == "ff":
        x, wg, wu, wd = inputs
        gate = x @ wg
        return (gate * torch.sigmoid(gate) * (x @ wu)) @ wd
    q, k, v, pos, pos_k, slope = inputs
    return _plain_attention(s, q, k, v, pos, pos_k, slope)


def _own(s, op, inputs):
    from equitorch_amd.nn import functional as F
    if op == "embed":
        return F.embedding(s["kind"], inputs[0], s["scale"])
    if op == "ff":
        return F.gated_feed_forward(*inputs)
    q, k, v, pos, pos_k, slope = inputs
    return F.segment_attention(q, k, v, s["plan"], pos=pos, slope=slope, pos_k=pos_k, cap=s["cap"], scale=s["scale"])


def _inputs(s):
    op = s["case"]["op"]
    if op == "embed":
        return [s["table"]]
    if op == "ff":
        return [s["x"], *s["w"]]
    return [*s["qkv"], s["pos"], s["pos_k"], s["slope"]]


def run(s):
    op, given = s["case"]["op"], _inputs(s)
    if s["case"]["pass"] == "forward":
        with torch.no_grad():
            if own:
                return _own(s, op, given)
            return _plain(s, op, [None if t is None else t.float() for t in given]).to(given[0].dtype)
    if own:
        out = _own(s, op, given)
        return (out, *torch.autograd.grad(out, [t for t in given if t is not None], s["ct"]))
    wide = [None if t is None else t.detach().float().requires_grad_(True) for t in given]
    out = _plain(s, op, wide)
    grads = torch.autograd.grad(out, [t for t in wide if t is not None], s["ct"].float())
    return (out.detach().to(given[0].dtype), *[g.to(t.dtype) for g, t in zip(grads, [t for t in given if t is not None])])


# ---- what a pass cannot do without ----------------------------------------------------------------------------
def work(case):
    b, step = (4 if case["dtype"] == "f32" else 2), case["pass"] == "step"
    if case["op"] == "embed":
        n, c = case["rows"], case["channels"]
        table = min(case["kinds"], n) * c * b
        nbytes = 8 * n + table + n * c * b
        if step:
            nbytes += 8 * n + n * c * b + case["kinds"] * c * b
        return {"bytes": nbytes, "flops": n * c * (2 if step else 1)}
    if case["op"] == "ff":
        n, c, h = case["rows"], case["channels"], case["hidden"]
        weights, row = 3 * c * h * b, n * c * b
        if step:   # x, ct, weights in; y, the gradients of x and of the weights out
            return {"bytes": 4 * row + 2 * weights, "flops": 18.0 * n * c * h}
        return {"bytes": 2 * row + weights, "flops": 6.0 * n * c * h}
    len_q, len_k = _sizes(case)
    nq, nk, hq, hk, d = sum(len_q), sum(len_k), case["heads"], case["kv_heads"], case["dim"]
    pairs = sum(i * j for i, j in zip(len_q, len_k))
    pos = 12 * (nk + (nq if case["queries"] == "one" else 0)) if case["bias"] else 0
    nbytes = (2 * nq * hq + 2 * nk * hk) * d * b + pos
    if step:       # the gradient of the output in; the gradients of q, k, v and the positions out
        nbytes += (2 * nq * hq + 2 * nk * hk) * d * b + pos
    return {"bytes": nbytes, "flops": (14.0 if step else 4.0) * pairs * hq * d}


# ---- 64-bit results -------------------------------------------------------------------------------------------
def _exact_attention(s, ct):
    """Structure by structure and head by head, from the definition; the gradients by their formulas."""
    case = s["case"]
    q, k, v = (t.detach().double() for t in s["qkv"])
    pos = None if s["pos"] is None else s["pos"].detach().double()
    pos_k = pos if s["pos_k"] is None else s["pos_k"].detach().double()
    slope = None if s["slope"] is None else s["slope"].detach().double()
    group, a, cap = case["heads"] // case["kv_heads"], s["scale"], s["cap"]
    out, gq, gk, gv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    g_pos = None if pos is None else torch.zeros_like(pos)
    g_pos_k = None if pos is None else torch.zeros_like(pos_k)
    g_slope = None if slope is None else torch.zeros_like(slope)
    len_q, len_k = _sizes(case)
    q0 = k0 = 0
    for lq, lk in zip(len_q, len_k):
        rq, rk = slice(q0, q0 + lq), slice(k0, k0 + lk)
        q0, k0 = q0 + lq, k0 + lk
        if lq == 0 or lk == 0:
            continue
        if pos is not None:
            delta = pos[rq, None] - pos_k[None, rk]
            dist = torch.linalg.vector_norm(delta, dim=-1)
            unit = delta / dist.masked_fill(dist == 0, 1.0)[..., None]
            along = torch.zeros_like(dist)
            del delta
        for h in range(case["heads"]):
            hk = h // group
            z = (q[rq, h] @ k[rk, hk].T) * a
            t = torch.tanh(z / cap) if cap else None
            z = cap * t if cap else z
            if pos is not None:
                z = z - slope[h] * dist
            p = torch.softmax(z, dim=1)
            out[rq, h] = p @ v[rk, hk]
            if ct is None:
                continue
            g = ct[rq, h]
            gv[rk, hk] += p.T @ g
            gz = g @ v[rk, hk].T
            gz = p * (gz - (p * gz).sum(1, keepdim=True))
            if pos is not None:
                g_slope[h] -= (gz * dist).sum()
                along -= slope[h] * gz
            if cap:
                gz = gz * (1 - t * t)
            gq[rq, h] = a * (gz @ k[rk, hk])
            gk[rk, hk] += a * (gz.T @ q[rq, h])
        if ct is not None and pos is not None:
            pull = along[..., None] * unit
            g_pos[rq] += pull.sum(1)
            g_pos_k[rk] -= pull.sum(0)
    if ct is None:
        return out
    if pos is None:
        return out, gq, gk, gv
    if s["pos_k"] is None:
        return out, gq, gk, gv, g_pos + g_pos_k, g_slope
    return out, gq, gk, gv, g_pos, g_pos_k, g_slope


def exact(case, seed):
    s = _tensors(case, seed)
    with torch.no_grad():
        ct = s["ct"].double() if "ct" in s else None
        if case["op"] == "attn":
            return _exact_attention(s, ct)
        if case["op"] == "embed":
            table, kind = s["table"].detach().double(), s["kind"]
            out = table.index_select(0, kind) * s["scale"]
            if ct is None:
                return out
            return out, torch.zeros_like(table).index_add_(0, kind, ct * s["scale"])
        x, (wg, wu, wd) = s["x"].detach().double(), (t.detach().double() for t in s["w"])
        u, r = x @ wg, x @ wu
        sig = 1 / (1 + torch.exp(-u))
        mid = u * sig * r
        y = mid @ wd
        if ct is None:
            return y
        g_mid = ct @ wd.T
        g_u, g_r = g_mid * r * (sig + u * sig * (1 - sig)), g_mid * u * sig
        return y, g_u @ wg.T + g_r @ wu.T, x.T @ g_u, x.T @ g_r, mid.T @ ct
