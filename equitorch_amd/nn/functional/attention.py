"""Attention among the nodes of a structure, on invariant channels.

    s_ij = cap tanh(scale q_i.k_j / cap) - slope_h |r_i - r_j|,      out_i = sum_j softmax_j(s_ij) v_j

over the keys ``j`` of the query's own structure.  The structures of a batch lie one after the other, and
:class:`AttentionPlan` holds where they begin; ``cgtp_attn_forward`` and ``cgtp_attn_backward`` walk each structure's own
keys only, never a padded or masked square."""
import ctypes as C
from typing import Optional

import numpy as np
import torch
from torch import Tensor
from torch.autograd import Function

from ... import _lib, _shim
from ..._lib import AttnArgs, CgtpError
from ._higher_order import higher_order

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_MOST = 2 ** 31 - 1024          # the kernels count keys and rows in 32 bits, up to four tiles beyond the last one
_BLOCK = 64                     # keys (rows) of a tile: pieces of a structure begin at multiples of it
_PIECE = 256                    # keys (rows) of a piece at least
_LEAST = 64                     # the same where tiles are few
_SMALL = 256                    # tiles of 32 rows that leave wavefronts idle: four for each make one for each SIMD
_WAVES = 4096                   # wavefronts wanted where structures can be cut into pieces: four for each SIMD


def _lengths(ptr: Tensor, name: str) -> np.ndarray:
    if ptr.ndim != 1 or ptr.dtype != torch.int64 or ptr.shape[0] < 1:
        raise CgtpError(f"{name} must be a 1-d int64 tensor of S + 1 offsets, got {ptr.dtype} {tuple(ptr.shape)}")
    p = ptr.detach().cpu().numpy()
    lengths = np.diff(p)
    if p[0] != 0 or (lengths < 0).any() or p[-1] >= _MOST:
        raise CgtpError(f"{name} must start at 0, never descend and stay below 2^31 - 1024")
    return lengths


class _Items:
    """Tables of one pass for the kernels: tiles of ``tile`` rows of every structure, each against the columns of its
    structure, or against a piece of them where there are too few tiles to occupy the GPU."""

    def __init__(self, rows: np.ndarray, cols: np.ndarray, tile: int, heads: int, waves: int, least: int = _PIECE, wanted: int = _WAVES):
        tiles = -(-rows // tile)
        s = np.repeat(np.arange(len(rows)), tiles)                             # structure of every tile
        first_tile = np.cumsum(tiles) - tiles
        begin = (np.arange(len(s)) - first_tile[s]) * tile
        end = np.minimum(begin + tile, rows[s])
        want = max(1, -(-wanted // (waves * heads * max(1, len(s)))))          # pieces of a tile where all are alike
        # Where that leaves a tile pieces of more than four times the share of the batch's columns that keeps a wavefront as busy as the
        # others, it gets pieces of such a share: it would run alone at the end (64 readouts, 63 over 300 keys and one over
        # 100000, 8 heads of 32, fp32: forward 1720 us in one piece, 73 so).
        share = max(1, -(-int(cols[s].sum()) * heads * waves // wanted))
        want = np.where(cols[s] > 4 * share * want, -(-cols[s] // share), want)
        pieces = np.clip(cols[s] // least, 1, want)
        step = -(-(-(-cols[s] // pieces)) // _BLOCK) * _BLOCK                  # columns of a piece
        pieces = np.maximum(1, -(-cols[s] // np.maximum(step, 1)))
        t = np.repeat(np.arange(len(s)), pieces)                               # tile of every piece
        first_piece = np.cumsum(pieces) - pieces
        place = np.arange(len(t)) - first_piece[t]
        cut = pieces > 1
        slot = np.cumsum(cut[t]) - 1
        self.structure, self.tile_structure, self.cut = s[t], s, cut
        self.begin, self.end, self.tile_begin, self.tile_end = begin[t], end[t], begin, end
        self.col_begin = place * step[t]
        self.col_end = np.minimum(self.col_begin + step[t], cols[s[t]])
        self.slot = np.where(cut[t], slot, -1)
        self.place = place
        self.first_slot = np.where(cut, self.slot[np.minimum(first_piece, max(0, len(t) - 1))], -1) if len(t) else cut
        self.pieces, self.slots = pieces, int(cut[t].sum())
        # the most work first, so that the last workgroups to start are short ones
        self.order = np.argsort(-(self.col_end - self.col_begin), kind="stable")


def _table(columns, order, device) -> Optional[Tensor]:
    table = np.stack([np.asarray(c) for c in columns], axis=1).astype(np.int32)
    if order is not None:
        table = table[order]
    return torch.from_numpy(np.ascontiguousarray(table)).to(device) if len(table) else None


class _Tables:
    def __init__(self, plan: "AttentionPlan", group: int, heads: int):
        cols, rows = plan.len_k, plan.len_q * group
        if rows.sum() >= _MOST:
            raise CgtpError("queries times query heads of a head of keys must stay below 2^31 - 1024")
        start_q, start_k = np.cumsum(plan.len_q) - plan.len_q, np.cumsum(cols) - cols
        # Tiles of 128 rows share a tile of keys among four wavefronts; tiles of 32 rows waste less of a short structure.  Few
        # rows against many keys (a readout), or so few tiles that the GPU is idle otherwise: four wavefronts share out the
        # keys of a tile of 32 rows (8 structures of 510 nodes, a head of 48, fp32: forward 48 -> 22 us; but 376 tiles of 2
        # structures of 3000 nodes 144 so, 127 by 128).
        self.wide_q, self.wide_k = int(_wide(rows)), int(_wide(cols))
        tiles = int((-(-rows // 32)).sum())
        if not self.wide_q and int(cols.sum()) >= 96 * tiles or 0 < tiles * heads <= _SMALL and int(cols.max()) > 32:
            self.wide_q = 2
        # Two for each SIMD, all at once, where there are few rows: more pieces take another turn and a longer join (one query of 8
        # heads on 2 over 200003 keys, bf16: 38 us with four, 31 so).
        q = _Items(rows, cols, 128 if self.wide_q == 1 else 32, heads, 4 if self.wide_q else 1,
                   wanted=_WAVES // 2 if self.wide_q == 2 else _WAVES)
        # The gradient of keys and values likewise, by short pieces of the rows (151 nodes, 4 query heads on one of 128, fp32: step
        # 203 -> 116 us, 8 structures of 510 nodes, a head of 48, 211 -> 104).
        few = int((-(-cols // 32)).sum()) * heads <= _SMALL
        self.wide_k = int(self.wide_k and not few)
        k = _Items(cols, rows, 128 if self.wide_k else 32, heads, 4 if self.wide_k else 1, _LEAST if few else _PIECE)
        zero = np.zeros_like(q.begin)
        at = start_k[q.structure]
        self.q_items = _table((start_q[q.structure], q.begin, q.end, at + q.col_begin, at + q.col_end, q.slot, q.place, zero),
                              q.order, plan.device)
        cut = q.cut
        zero = np.zeros_like(q.tile_begin)[cut]
        s = q.tile_structure[cut]
        self.q_joins = _table((start_q[s], q.tile_begin[cut], q.tile_end[cut], zero, zero, zero, q.first_slot[cut],
                               q.pieces[cut]), None, plan.device)
        at = start_k[k.structure]
        zero = np.zeros_like(k.begin)
        self.k_items = _table((start_q[k.structure], k.col_begin, k.col_end, at + k.begin, at + k.end, k.slot, k.place, zero),
                              k.order, plan.device)
        cut = k.cut
        zero = np.zeros_like(k.tile_begin)[cut]
        s = k.tile_structure[cut]
        self.k_joins = _table((start_q[s], zero, zero, start_k[s] + k.tile_begin[cut], start_k[s] + k.tile_end[cut], zero,
                               k.first_slot[cut], k.pieces[cut]), None, plan.device)
        self.q_slots, self.k_slots = q.slots, k.slots
        self.stream = _stream_of(plan.device)

    def put(self, a: AttnArgs) -> None:
        _record(self.stream, self.q_items, self.q_joins, self.k_items, self.k_joins)
        for name in ("q_items", "q_joins", "k_items", "k_joins"):
            t = getattr(self, name)
            setattr(a, name, _lib.ptr(t))
            setattr(a, "n_" + name, 0 if t is None else t.shape[0])
        a.n_q_slots, a.n_k_slots, a.wide_q, a.wide_k = self.q_slots, self.k_slots, self.wide_q, self.wide_k


def _stream_of(device) -> int:
    return _lib.stream_ptr(device) if device.type == "cuda" else 0


def _record(stream: int, *tensors: Optional[Tensor]) -> None:
    """What a plan holds is read on the current stream: where that is not the stream of its memory, ``stream``, the memory is not
    handed out again before what is queued here is done."""
    for t in tensors:
        if t is not None and t.is_cuda and _stream_of(t.device) != stream:
            t.record_stream(torch.cuda.current_stream(t.device))


def _wide(n: np.ndarray) -> bool:
    """Whether tiles of 128 cover the structures with at most a quarter more rows than tiles of 32."""
    return int((-(-n // 128) * 128).sum()) * 4 <= int((-(-n // 32) * 32).sum()) * 5


class AttentionPlan:
    """Where the structures of a batch begin: ``ptr`` int64 ``(S + 1,)``, ``ptr[s] .. ptr[s + 1]`` the nodes of structure
    ``s``, and ``ptr_k`` the same for the keys where queries and keys are different nodes (a readout: one query for each
    structure).  Structures may be empty, on either side.  Built once for a batch (it reads ``ptr`` on the host), used by
    every layer; the kernels' tables are made on first use for each number of heads and kept with it (a graph is captured after
    that, and reads them for as long as it is replayed).  A plan may be used, and dropped, on any stream."""

    def __init__(self, ptr: Tensor, ptr_k: Optional[Tensor] = None):
        self.device = ptr.device
        self.len_q = _lengths(ptr, "ptr")
        self.len_k = self.len_q if ptr_k is None else _lengths(ptr_k, "ptr_k")
        if len(self.len_k) != len(self.len_q):
            raise CgtpError(f"ptr has {len(self.len_q)} structures, ptr_k {len(self.len_k)}")
        if ptr_k is not None and ptr_k.device != ptr.device:
            raise CgtpError(f"ptr is on {ptr.device}, ptr_k on {ptr_k.device}")
        self.num_structures = len(self.len_q)
        self.num_queries, self.num_keys = int(self.len_q.sum()), int(self.len_k.sum())
        self._tables, self._handles = {}, {}
        self._buckets = _Buckets(self.len_q, self.len_k, self.device)

    @classmethod
    def from_batch(cls, batch: Tensor, num_structures: Optional[int] = None) -> "AttentionPlan":
        """From the structure of every node, ascending."""
        if batch.ndim != 1 or batch.dtype != torch.int64:
            raise CgtpError(f"batch must be a 1-d int64 tensor, got {batch.dtype} {tuple(batch.shape)}")
        b = batch.detach().cpu().numpy()
        n = int(num_structures) if num_structures is not None else (int(b[-1]) + 1 if len(b) else 0)
        if len(b) and ((np.diff(b) < 0).any() or b[0] < 0 or b[-1] >= n):
            raise CgtpError(f"batch must ascend within 0 .. {n - 1}")
        ptr = np.concatenate([[0], np.cumsum(np.bincount(b, minlength=n))]).astype(np.int64)
        return cls(torch.from_numpy(ptr).to(batch.device))

    def tables(self, group: int, heads: int) -> _Tables:
        """For ``heads`` heads of keys with ``group`` query heads each."""
        key = (group, heads)
        if key not in self._tables:
            self._tables[key] = _Tables(self, group, heads)
        return self._tables[key]

    def handle(self, mod, group: int, heads: int):
        """The extension's copy of the tables, and the tensor expression its node evaluates under gradient mode."""
        key = (group, heads)
        if key not in self._handles:
            t, buckets = self.tables(group, heads), self._buckets
            h = mod.AttnHandle(t.q_items, t.q_joins, t.k_items, t.k_joins, t.q_slots, t.k_slots, t.wide_q, t.wide_k, t.stream)
            # holds the buckets, not the plan: the node keeps it for as long as it lives itself
            h.set_fallback(lambda g, inputs, need, scale, cap: higher_order(_of_buckets(buckets, scale, cap), inputs, need, g))
            self._handles[key] = h
        return self._handles[key]


class _Buckets:
    """Structures of similar length together, padded to the longest of each bucket, for the tensor expression; made on first
    use."""

    def __init__(self, len_q: np.ndarray, len_k: np.ndarray, device):
        self.len_q, self.len_k, self.device, self._made = len_q, len_k, device, None

    def get(self):
        """``(rows_q, keep_q, rows_k, keep_k)`` per bucket and the order that sorts the buckets' queries."""
        if self._made is None:
            start_q, start_k = np.cumsum(self.len_q) - self.len_q, np.cumsum(self.len_k) - self.len_k
            groups = {}
            for s in np.flatnonzero(self.len_q):
                groups.setdefault((int(self.len_q[s]).bit_length(), int(self.len_k[s]).bit_length()), []).append(s)
            out, order = [], []
            for members in groups.values():
                m = np.asarray(members)
                index = []
                for start, n in ((start_q[m], self.len_q[m]), (start_k[m], self.len_k[m])):
                    col = np.arange(max(1, n.max()))[None]
                    keep = col < n[:, None]
                    index += [np.where(keep, start[:, None] + col, 0), keep]
                order.append(index[0][index[1]])
                out.append(tuple(torch.from_numpy(i).to(self.device) for i in index))
            order = np.concatenate(order) if order else np.zeros(0, dtype=np.int64)
            self._made = (out, torch.from_numpy(np.argsort(order)).to(self.device))
            self._stream = _stream_of(self.device)
        _record(self._stream, self._made[1], *(t for bucket in self._made[0] for t in bucket))
        return self._made


def _of_buckets(buckets: _Buckets, scale: float, cap: float):
    def expression(q, k, v, pos_q, pos_k, slope):
        return _expression(q, k, v, pos_q, pos_q if pos_k is None else pos_k, slope, buckets, scale, cap)
    return expression


def _expression(q, k, v, pos_q, pos_k, slope, padded: _Buckets, scale: float, cap: float):
    """The same result as a tensor expression on padded buckets of structures, which autograd differentiates to any order
    (in 32 bits)."""
    dtype, group = q.dtype, q.shape[1] // k.shape[1]
    nothing = None
    if k.shape[0] == 0 or not padded.len_q.any():          # some operands are not read: their gradients are zeros all the same
        nothing = sum(t[:0].float().sum() for t in (q, k, v, pos_q, pos_k, slope) if t is not None)
    if k.shape[0] == 0:                     # no keys at all: something to point at; nothing of it is kept
        k, v = k.new_zeros((1, *k.shape[1:])), v.new_zeros((1, *v.shape[1:]))
        pos_k = None if pos_k is None else pos_k.new_zeros((1, 3))
    outs, (buckets, order) = [], padded.get()
    for rows_q, keep_q, rows_k, keep_k in buckets:
        qb = q[rows_q].float().masked_fill(~keep_q[:, :, None, None], 0.0).transpose(1, 2)
        # padding points at some node: what that holds may not reach a result, not even as a zero times an infinity
        kb, vb = (t[rows_k].float().masked_fill(~keep_k[:, :, None, None], 0.0).transpose(1, 2)
                  .repeat_interleave(group, dim=1) for t in (k, v))
        s = torch.matmul(qb, kb.transpose(2, 3).contiguous()) * scale
        if cap > 0:
            s = cap * torch.tanh(s / cap)
        if slope is not None:
            diff = pos_q[rows_q].masked_fill(~keep_q[:, :, None], 0.0)[:, :, None] - pos_k[rows_k].masked_fill(~keep_k[:, :, None], 0.0)[:, None]
            d2 = (diff * diff).sum(-1).clamp(max=3e38)       # where fp32 ends: -1e19 times the slope for its score, and no inf * 0
            s = s - slope[:, None, None] * torch.where(d2 > 0, torch.where(d2 > 0, d2, torch.ones_like(d2)).sqrt(),
                                                       torch.zeros_like(d2))[:, None]
        s = s.masked_fill(~keep_k[:, None, None], -torch.inf)
        top = s.amax(-1, keepdim=True).detach()
        p = torch.exp(s - torch.where(top > -torch.inf, top, torch.zeros_like(top)))
        total = p.sum(-1, keepdim=True)
        out = torch.matmul(p, vb) / torch.where(total > 0, total, torch.ones_like(total))
        outs.append(out.transpose(1, 2)[keep_q])
    out = torch.cat(outs)[order].to(dtype) if outs else q * 0.0
    return out if nothing is None else out + nothing


def _args(q, k, v, pos_q, pos_k, slope, plan, scale, cap) -> AttnArgs:
    a = AttnArgs()
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_node, a.q_head = q.stride(0), q.stride(1)
    a.k_node, a.k_head = k.stride(0), k.stride(1)
    a.v_node, a.v_head = v.stride(0), v.stride(1)
    a.pos_q, a.pos_k, a.slope = _lib.ptr(pos_q), _lib.ptr(pos_k), _lib.ptr(slope)
    a.n_q, a.n_k, a.h_q, a.h_kv, a.dim = q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2]
    a.dtype, a.scale, a.cap = _lib.dtype_code(q.dtype), scale, cap
    plan.tables(a.h_q // a.h_kv, a.h_kv).put(a)
    return a


def _forward(q, k, v, pos_q, pos_k, slope, plan, scale, cap, keep):
    """``(out, lse)``; lse, which a backward reads, is None unless ``keep``."""
    a = _args(q, k, v, pos_q, pos_k, slope, plan, scale, cap)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if keep else None
    a.out, a.lse = out.data_ptr(), _lib.ptr(lse)
    nbytes = _lib.lib.cgtp_attn_workspace_bytes(C.byref(a), 0)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    a.workspace = _lib.ptr(ws)
    _lib.check(_lib.lib.cgtp_attn_forward(C.byref(a), _lib.stream_ptr(q.device)), "cgtp_attn_forward")
    return out, lse


class _SegmentAttention(Function):
    """``pos_k`` None: the queries' positions are the keys' too, and their gradient is the sum over both."""

    @staticmethod
    def forward(ctx, q, k, v, pos_q, pos_k, slope, plan, scale, cap):
        out, lse = _forward(q, k, v, pos_q, pos_q if pos_k is None else pos_k, slope, plan, scale, cap, True)
        ctx.save_for_backward(q, k, v, pos_q, pos_k, slope, out, lse)
        ctx.plan, ctx.scale, ctx.cap = plan, scale, cap
        return out

    @staticmethod
    def backward(ctx, g):
        q, k, v, pos_q, pos_k, slope, out, lse = ctx.saved_tensors
        need, plan, scale, cap = ctx.needs_input_grad[:6], ctx.plan, ctx.scale, ctx.cap
        if torch.is_grad_enabled():
            expression = _of_buckets(plan._buckets, scale, cap)
            return (*higher_order(expression, (q, k, v, pos_q, pos_k, slope), need, g), None, None, None)
        g = g.contiguous()
        g = g if g.data_ptr() % 16 == 0 else g.clone()
        a = _args(q, k, v, pos_q, pos_q if pos_k is None else pos_k, slope, plan, scale, cap)
        a.out, a.lse, a.grad_out = out.data_ptr(), lse.data_ptr(), g.data_ptr()
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if n else None
                 for t, n in zip((q, k, v, pos_q, pos_k, slope), need)]
        a.grad_q, a.grad_k, a.grad_v, a.grad_pos_q, a.grad_pos_k, a.grad_slope = (_lib.ptr(t) for t in grads)
        a.same_pos = pos_k is None
        ws = torch.empty(_lib.lib.cgtp_attn_workspace_bytes(C.byref(a), 1), dtype=torch.uint8, device=q.device)
        a.workspace = ws.data_ptr()
        _lib.check(_lib.lib.cgtp_attn_backward(C.byref(a), _lib.stream_ptr(q.device)), "cgtp_attn_backward")
        return (*grads, None, None, None)


def _check(q, k, v, plan, pos, slope, pos_k):
    _lib.require_gpu(q, k, v, pos, slope, pos_k)
    if q.ndim != 3 or k.ndim != 3 or v.shape != k.shape or q.shape[2] != k.shape[2]:
        raise CgtpError(f"q must be (N_q, H_q, D), k and v (N_k, H_kv, D), got {tuple(q.shape)}, {tuple(k.shape)}, "
                        f"{tuple(v.shape)}")
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    if hk < 1 or hq < 1 or hq % hk or not 1 <= d <= 128:
        raise CgtpError(f"query heads must be a multiple of key heads and D 1 .. 128, got {hq}, {hk}, {d}")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise CgtpError(f"q, k and v must be fp32, bf16 or fp16, all of one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    if plan.num_queries != q.shape[0] or plan.num_keys != k.shape[0]:
        raise CgtpError(f"plan was built for {plan.num_queries} queries and {plan.num_keys} keys, got {q.shape[0]} and "
                        f"{k.shape[0]}")
    if any(t is not None and t.device != plan.device for t in (q, k, v, pos, slope, pos_k)):
        raise CgtpError(f"operands must be on the plan's device, {plan.device}")
    if slope is None:
        if pos is not None or pos_k is not None:
            raise CgtpError("positions are read with a slope only")
        return
    if pos is None or (pos_k is None and plan.len_k is not plan.len_q):
        raise CgtpError("a slope needs the queries' positions, and the keys' where these are other nodes")
    for name, t, shape in (("pos", pos, (q.shape[0], 3)), ("pos_k", pos_k, (k.shape[0], 3)), ("slope", slope, (hq,))):
        if t is not None and (tuple(t.shape) != shape or t.dtype != torch.float32):
            raise CgtpError(f"{name} must be fp32 {shape}, got {t.dtype} {tuple(t.shape)}")


def segment_attention(q: Tensor, k: Tensor, v: Tensor, plan: AttentionPlan, pos: Optional[Tensor] = None,
                      slope: Optional[Tensor] = None, pos_k: Optional[Tensor] = None, cap: Optional[float] = None,
                      scale: Optional[float] = None) -> Tensor:
    """Softmax attention of every query over the keys of its own structure: ``q`` ``(N_q, H_q, D)``, ``k`` and ``v``
    ``(N_k, H_kv, D)`` in fp32, bf16 or fp16, ``H_q`` a multiple of ``H_kv`` (neighbouring query heads share a head of keys
    and values), ``D`` up to 128; slices of a common projection are read where they are.  ``scale`` is ``D ** -0.5`` unless
    given.

    ``cap``: scores are ``cap * tanh(score / cap)``.  ``slope`` fp32 ``(H_q,)`` and ``pos`` fp32 ``(N_q, 3)`` (``pos_k``
    ``(N_k, 3)`` where the keys are other nodes): ``slope_h`` times the distance is taken off the score.  The gradient of a
    distance of zero is zero.  A query without keys, or whose scores are all -inf, gets zeros, and so do its gradients; where only
    some are, because of infinities in those keys, its own gradient is a sum with 0 * inf in it (in gradient mode in either case).

    Statistics and sums are in 32 bits; in 16-bit types the probabilities and the scores' gradients are rounded to the type
    as operands of the next product (in fp16 scaled into its range first).  Results do not depend on timing; differentiable to any order, beyond the first
    through a tensor expression that holds the scores of every structure in memory."""
    q, k, v = _lib.of_one_type(q, k, v)
    _check(q, k, v, plan, pos, slope, pos_k)
    cap = 0.0 if cap is None else float(cap)
    if not 0.0 <= cap < float("inf"):
        raise CgtpError(f"cap must be positive and finite (or None), got {cap}")
    if cap > 0.0:
        cap = min(max(cap, 2.0 ** -100), 2.0 ** 127)      # as a float neither zero, which is no cap, nor infinite
    scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    q, k, v = (t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous() for t in (q, k, v))
    pos, pos_k, slope = (None if t is None else t.contiguous() for t in (pos, pos_k, slope))
    keep = (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, pos, pos_k, slope))) \
        or _lib.forward_mode()
    mod = _shim.module()
    if mod is not None:
        handle = plan.handle(mod, q.shape[1] // k.shape[1], k.shape[1])
        return mod.attn(q, k, v, pos, pos_k, slope, handle, scale, cap, keep)
    if keep:
        return _SegmentAttention.apply(q, k, v, pos, pos_k, slope, plan, scale, cap)
    return _forward(q, k, v, pos, pos if pos_k is None else pos_k, slope, plan, scale, cap, False)[0]
