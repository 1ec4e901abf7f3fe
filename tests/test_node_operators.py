"""Embedding, attention and gated feed-forward on invariant channels without a GPU: layouts of the argument structs, the
codes of refused calls, and the tables the attention's kernels walk."""
import ctypes as C

import numpy as np
import pytest
import torch

from equitorch_amd import _lib
from equitorch_amd._lib import AttnArgs, CgtpError, GffArgs

NULL, SHAPE, ALIGN, DTYPE, CONFIG, WORKSPACE = 1, 2, 3, 4, 5, 8


class _Item(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("node", "row_begin", "row_end", "k_begin", "k_end", "slot", "first", "count")]


@pytest.mark.parametrize("which,cls", [(17, GffArgs), (18, AttnArgs), (19, _Item)])
def test_struct_layouts(which, cls):
    n = _lib.lib.cgtp_abi_layout(which, None, 0)
    assert n == 1 + len(cls._fields_)
    buf = (C.c_int64 * n)()
    assert _lib.lib.cgtp_abi_layout(which, buf, n) == n
    assert list(buf) == [C.sizeof(cls)] + [getattr(cls, name).offset for name, _ in cls._fields_]


def test_embedding_codes():
    lib, p = _lib.lib, 4096
    assert lib.cgtp_embed_forward(p, p, p, 5, 0, 8, 1.0, 0, None) == SHAPE
    assert lib.cgtp_embed_forward(p, p, p, -1, 3, 8, 1.0, 0, None) == SHAPE
    assert lib.cgtp_embed_forward(p, p, p, 5, 3, 8, 1.0, 9, None) == DTYPE
    assert lib.cgtp_embed_forward(None, p, p, 5, 3, 8, 1.0, 0, None) == NULL
    assert lib.cgtp_embed_forward(None, None, None, 0, 3, 8, 1.0, 0, None) == 0
    assert lib.cgtp_embed_backward(p, p, None, p, 5, 3, 8, 1.0, 0, None) == NULL
    assert lib.cgtp_embed_backward(p, p, p, None, 5, 3, 8, 1.0, 0, None) == WORKSPACE
    assert lib.cgtp_embed_workspace_bytes(0, 3, 8, 0) == lib.cgtp_embed_workspace_bytes(5, 3, 8, 9) == 0
    assert lib.cgtp_embed_workspace_bytes(1000, 100, 64, 0) > 8 * 1000


def _gff(**changed):
    a = GffArgs()
    for name in ("x", "w_gate", "w_up", "w_down", "gate", "up", "mid", "out", "grad_out", "grad_gate", "grad_up"):
        setattr(a, name, 4096)
    a.n_rows, a.c_in, a.hidden, a.c_out = 5, 8, 16, 8
    for name, value in changed.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changed,forward,backward", [
    ({"dtype": 1}, DTYPE, DTYPE), ({"c_in": 0}, SHAPE, SHAPE), ({"hidden": 1 << 20}, SHAPE, SHAPE), ({"n_rows": -1}, SHAPE, SHAPE),
    ({"activation": 3}, CONFIG, CONFIG), ({"w_up": None}, NULL, NULL), ({"x": None}, NULL, NULL), ({"out": None}, NULL, 0),
    ({"gate": None}, NULL, NULL), ({"grad_out": None, "n_rows": 0}, 0, 0), ({"mid": None}, NULL, NULL)])
def test_feed_forward_codes(changed, forward, backward):
    a = _gff(**changed)
    assert _lib.lib.cgtp_gff_forward(C.byref(a), None) == forward
    assert _lib.lib.cgtp_gff_forward(None, None) == NULL
    if backward:
        assert _lib.lib.cgtp_gff_backward(C.byref(a), None) == backward


def test_feed_forward_workspace():
    a = _gff(n_rows=100000, grad_w_gate=4096)
    assert _lib.lib.cgtp_gff_workspace_bytes(C.byref(a), 1) > 0
    assert _lib.lib.cgtp_gff_backward(C.byref(a), None) == WORKSPACE


def test_feed_forward_copies_rows_of_large_calls():
    def need(n_rows, c, backward):
        a = _gff(n_rows=n_rows, c_in=c, hidden=250, c_out=8, dtype=2, grad_x=4096)
        return _lib.lib.cgtp_gff_workspace_bytes(C.byref(a), backward)
    rows, weights = 20000, (15 + 15) * 256 + 250 * 8
    assert need(rows, 15, 0) == 2 * (rows * 16 + weights)
    assert need(rows, 15, 1) >= 2 * (rows * 16 + weights + rows * 8)
    assert need(100, 15, 0) == 0
    for name in ("mid", "gate"):
        assert _lib.lib.cgtp_gff_forward(C.byref(_gff(**{name: 4098})), None) == ALIGN
    for name in ("mid", "up", "grad_gate", "grad_up"):
        assert _lib.lib.cgtp_gff_backward(C.byref(_gff(**{name: 4098})), None) == ALIGN


def _attn(**changed):
    a = AttnArgs()
    for name in ("q", "k", "v", "out", "lse", "q_items", "k_items", "grad_out", "pos_q", "pos_k", "slope", "workspace"):
        setattr(a, name, 4096)
    a.n_q, a.n_k, a.h_q, a.h_kv, a.dim, a.n_q_items, a.n_k_items = 4, 4, 2, 1, 16, 1, 1
    for name, value in changed.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changed,status", [
    ({"dtype": 1}, DTYPE), ({"dim": 129}, SHAPE), ({"dim": 0}, SHAPE), ({"h_q": 3, "h_kv": 2}, SHAPE), ({"h_kv": 0}, SHAPE),
    ({"n_q": -1}, SHAPE), ({"n_k": 1 << 31}, SHAPE), ({"n_q": 1 << 30, "h_q": 4}, SHAPE), ({"n_q_items": -1}, SHAPE),
    ({"n_q_items": 1 << 24}, SHAPE), ({"n_q_joins": 1 << 22}, SHAPE), ({"q": None}, NULL), ({"v": None}, NULL), ({"out": None}, NULL),
    ({"q_items": None}, NULL), ({"pos_k": None}, NULL)])
def test_attention_codes(changed, status):
    a = _attn(**changed)
    assert _lib.lib.cgtp_attn_forward(C.byref(a), None) == status
    assert _lib.lib.cgtp_attn_backward(C.byref(a), None) == status
    assert _lib.lib.cgtp_attn_workspace_bytes(C.byref(a), 1) == 0


def test_attention_codes_of_one_direction():
    lib = _lib.lib
    assert lib.cgtp_attn_forward(None, None) == NULL
    assert lib.cgtp_attn_forward(C.byref(_attn(n_q_slots=2, workspace=None)), None) == WORKSPACE
    assert lib.cgtp_attn_backward(C.byref(_attn(workspace=None)), None) == WORKSPACE
    assert lib.cgtp_attn_backward(C.byref(_attn(lse=None)), None) == NULL
    assert lib.cgtp_attn_backward(C.byref(_attn(k_items=None)), None) == NULL
    assert lib.cgtp_attn_forward(C.byref(_attn(workspace=4100)), None) == ALIGN
    assert lib.cgtp_attn_backward(C.byref(_attn(workspace=4100)), None) == ALIGN


def test_attention_copies_rows_that_are_not_whole():
    strides = dict(q_node=32, q_head=16, k_node=16, k_head=16, v_node=16, v_head=16)

    def need(backward=0, **changed):
        return _lib.lib.cgtp_attn_workspace_bytes(C.byref(_attn(**{**strides, "dtype": 2, **changed})), backward)
    kept = need(backward=1)
    assert need() == 0
    assert need(q=4098) == 256                               # 4 x 2 rows of 32 bytes
    assert need(k=4098) == need(v_node=17) == 256            # 4 rows
    assert need(q_node=-32) == need(q_node=1 << 30) == 256
    assert need(dim=15) == 3 * 256 and need(backward=1, dim=15) == kept + 4 * 256
    assert need(backward=1, grad_out=4098) == kept + 256
    for backward, launch in ((0, _lib.lib.cgtp_attn_forward), (1, _lib.lib.cgtp_attn_backward)):
        assert launch(C.byref(_attn(**{**strides, "dtype": 2, "q": 4098, "workspace": None})), None) == WORKSPACE


@pytest.mark.parametrize("len_q,len_k,group,heads", [
    ([3, 0, 7], None, 1, 8), ([700, 1], None, 2, 1), ([1, 1, 1, 0], [0, 70000, 300, 5], 4, 2), ([5000], [2], 1, 1),
    ([128] * 40, None, 1, 8), ([129, 300, 12], [1, 0, 9000], 3, 1), ([1], [1], 1, 1), ([0], [4], 1, 1), ([], None, 1, 1)])
def test_attention_tables_cover_every_pair_once(len_q, len_k, group, heads):
    from equitorch_amd.nn.functional import AttentionPlan
    ptr = lambda n: torch.tensor([0] + list(n)).cumsum(0)
    plan = AttentionPlan(ptr(len_q)) if len_k is None else AttentionPlan(ptr(len_q), ptr(len_k))
    len_k = len_q if len_k is None else len_k
    t = plan.tables(group, heads)
    start_q, start_k = ptr(len_q).tolist(), ptr(len_k).tolist()
    for items, joins, slots, tile, keyed in ((t.q_items, t.q_joins, t.q_slots, 128 if t.wide_q == 1 else 32, False),
                                             (t.k_items, t.k_joins, t.k_slots, 128 if t.wide_k else 32, True)):
        seen = {s: np.zeros((len_q[s] * group, len_k[s]), dtype=int) for s in range(len(len_q))}
        fixed = {s: np.zeros(len_k[s] if keyed else len_q[s] * group, dtype=int) for s in range(len(len_q))}
        of_slot = {}
        for node, r0, r1, k0, k1, slot, place, _ in ([] if items is None else items.tolist()):
            if keyed:
                s = next(i for i in range(len(len_k)) if start_k[i] <= k0 < k1 <= start_k[i + 1])
                assert k1 - k0 <= tile
            else:
                s = next(i for i in range(len(len_q)) if start_q[i] == node and len_q[i]
                         and (start_k[i] <= k0 <= k1 <= start_k[i + 1]))
                assert 0 <= r0 < r1 and r1 - r0 <= tile
            assert start_q[s] == node and r1 <= len_q[s] * group
            seen[s][r0:r1, k0 - start_k[s]:k1 - start_k[s]] += 1
            if place == 0:
                (fixed[s][k0 - start_k[s]:k1 - start_k[s]] if keyed else fixed[s][r0:r1])[:] += 1
            if slot >= 0:
                assert slot not in of_slot
                of_slot[slot] = (node, k0, k1) if keyed else (node, r0, r1)
        assert all((m == 1).all() for m in seen.values()) and all((m == 1).all() for m in fixed.values())
        assert sorted(of_slot) == list(range(slots))
        joined = []
        for node, r0, r1, k0, k1, _, first, count in ([] if joins is None else joins.tolist()):
            joined += range(first, first + count)
            assert count > 1 and all(of_slot[i] == ((node, k0, k1) if keyed else (node, r0, r1)) for i in range(first, first + count))
        assert sorted(joined) == list(range(slots))


def test_plan_refuses():
    from equitorch_amd.nn.functional import AttentionPlan
    for bad in (torch.tensor([1, 2]), torch.tensor([0, 3, 2]), torch.tensor([0, 1], dtype=torch.int32), torch.tensor([[0, 1]]),
                torch.tensor([], dtype=torch.int64)):
        with pytest.raises(CgtpError):
            AttentionPlan(bad)
    with pytest.raises(CgtpError):
        AttentionPlan(torch.tensor([0, 2]), torch.tensor([0, 2, 3]))
    for batch, n in ((torch.tensor([0, 2, 1]), 3), (torch.tensor([0, 3]), 3), (torch.tensor([-1, 0]), 2), (torch.tensor([0.0]), 1)):
        with pytest.raises(CgtpError):
            AttentionPlan.from_batch(batch, n)
    assert AttentionPlan.from_batch(torch.tensor([0, 0, 2]), 4).len_q.tolist() == [2, 0, 1, 0]


def test_cpu_tensors_are_refused():
    from equitorch_amd.nn.functional import AttentionPlan, embedding, gated_feed_forward, segment_attention
    x = torch.zeros(4, 8)
    with pytest.raises(CgtpError):
        embedding(torch.zeros(2, dtype=torch.int64), x)
    with pytest.raises(CgtpError):
        gated_feed_forward(x, x.T, x.T, x)
    q = x.view(4, 1, 8)
    with pytest.raises(CgtpError):
        segment_attention(q, q, q, AttentionPlan(torch.tensor([0, 4])))


def test_expression_of_the_attention_is_the_definition():
    """The tensor expression that gradients of higher order go through, against the definition, on the CPU."""
    from equitorch_amd.nn.functional import AttentionPlan
    from equitorch_amd.nn.functional.attention import _expression
    gen = torch.Generator().manual_seed(4)
    len_q, len_k = [3, 0, 5, 2, 1], [4, 2, 0, 9, 1]
    q, k, v = torch.randn(11, 4, 6, generator=gen), torch.randn(16, 2, 6, generator=gen), torch.randn(16, 2, 6, generator=gen)
    pos, pos_k, slope = torch.randn(11, 3, generator=gen), torch.randn(16, 3, generator=gen), torch.rand(4, generator=gen)
    pos_k[15] = pos[10]
    ptr = lambda n: torch.tensor([0] + n).cumsum(0)
    got = _expression(q, k, v, pos, pos_k, slope, AttentionPlan(ptr(len_q), ptr(len_k))._buckets, 0.4, 3.0)
    want, a, b = torch.zeros_like(q), 0, 0
    for lq, lk in zip(len_q, len_k):
        for h in range(4):
            if lq and lk:
                s = 3 * torch.tanh(q[a:a + lq, h] @ k[b:b + lk, h // 2].T * 0.4 / 3)
                s = s - slope[h] * torch.cdist(pos[a:a + lq], pos_k[b:b + lk], compute_mode="donot_use_mm_for_euclid_dist")
                want[a:a + lq, h] = torch.softmax(s, 1) @ v[b:b + lk, h // 2]
        a, b = a + lq, b + lk
    assert torch.allclose(got, want, rtol=0, atol=3e-6)


def test_feed_forward_limits_are_those_of_its_launches():
    """Refused from 2^21 tiles of 1024 rows by 64 hidden channels (128 of x and out) on, and by the widths; accepted below (the call then
    misses a buffer: nothing is launched)."""
    def code(n_rows, hidden, c_in=256, c_out=256):
        a = _gff(n_rows=n_rows, c_in=c_in, hidden=hidden, c_out=c_out, mid=None)
        codes = {_lib.lib.cgtp_gff_forward(C.byref(a), None), _lib.lib.cgtp_gff_backward(C.byref(a), None)}
        assert len(codes) == 1
        return codes.pop()
    assert code(1 << 24, 1024) == code(3 << 20, 8192) == code((1 << 27) - 1024, 1024) == NULL
    assert code(1 << 27, 1024) == code(1 << 24, 8192) == SHAPE
    assert code((1 << 31) - 1, 64, 128, 129) == SHAPE and code((1 << 30), 64, 128, 129) == SHAPE and code(1 << 30, 64, 128, 128) == NULL
    assert code(5, (1 << 17) - 1, (1 << 15) - 1, (1 << 15) - 1) == NULL
    assert code(5, 1 << 17) == code(5, 64, 1 << 15) == code(5, 64, 8, 1 << 15) == SHAPE


@pytest.mark.parametrize("len_q,len_k,group,heads,longest", [
    ([1] * 64, [100000] + [300] * 63, 1, 8, 8192), ([1] * 600, [300] * 300 + [100000] + [300] * 299, 2, 8, 20000),
    ([20] * 500 + [6000], None, 1, 2, 2048), ([0] * 40 + [2] * 40 + [1], [7] * 80 + [50000], 4, 1, 4096)])
def test_attention_tables_of_one_long_structure_among_many(len_q, len_k, group, heads, longest):
    """The long one's keys (rows) are cut by its own length, however many short ones there are, and every pair is still covered."""
    from equitorch_amd.nn.functional import AttentionPlan
    test_attention_tables_cover_every_pair_once(len_q, len_k, group, heads)
    ptr = lambda n: torch.tensor([0] + list(n)).cumsum(0)
    t = (AttentionPlan(ptr(len_q)) if len_k is None else AttentionPlan(ptr(len_q), ptr(len_k))).tables(group, heads)
    items = t.q_items
    assert int((items[:, 4] - items[:, 3]).max()) <= longest


@pytest.mark.parametrize("most", [2 ** 31 - 1024])
def test_attention_counts_stay_within_32_bits(most):
    """Kernels step through keys and rows by up to 256 at a time in 32 bits: the last ones that would step past the end are refused."""
    from equitorch_amd.nn.functional import AttentionPlan
    lib, steps = _lib.lib, 256
    assert most - 1 + 4 * steps < 2 ** 31
    # one more than the largest count is refused, the largest itself only misses a buffer (nothing is launched)
    for name in ("n_k", "n_q"):
        assert lib.cgtp_attn_forward(C.byref(_attn(**{name: most, "h_q": 1, "q_items": None})), None) == SHAPE
        assert lib.cgtp_attn_forward(C.byref(_attn(**{name: most - 1, "h_q": 1, "q_items": None})), None) == NULL
    assert lib.cgtp_attn_forward(C.byref(_attn(n_q=most // 2, h_q=2, q_items=None)), None) == SHAPE
    for bad in (most, 2 ** 31 - 1):
        with pytest.raises(CgtpError):
            AttentionPlan(torch.tensor([0, bad]))
    with pytest.raises(CgtpError):
        AttentionPlan(torch.tensor([0, most // 2]), torch.tensor([0, 4])).tables(2, 1)
