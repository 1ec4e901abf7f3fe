"""Saving and loading of AdamW's states without a GPU, on states that are made by hand."""
import pytest
import torch

from equitorch_amd._lib import CgtpError
from equitorch_amd.optim import BLOCK, AdamW

F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


def _params(*shapes, dtype=F32, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=gen).to(dtype)) for s in shapes]


def _states(opt, seed=1):
    """States such as two steps leave, of random numbers."""
    gen = torch.Generator().manual_seed(seed)
    for group in opt.param_groups:
        for p in group["params"]:
            rand = lambda: torch.empty_like(p, dtype=F32).copy_(torch.rand(p.shape, generator=gen))      # in the order of p's elements
            state = opt.state[p]
            state["step"] = torch.tensor(2.0)
            if group["state_bits"] == 32:
                state["exp_avg"], state["exp_avg_sq"] = rand(), rand()
            else:
                for name in ("exp_avg", "root_avg_sq"):
                    state[name] = (rand() * 400).to(E4M3)
                    state[name + "_scale"] = torch.rand(-(-p.numel() // BLOCK), generator=gen)
            if group["master"] and p.dtype != F32:
                state["master"] = rand()
    return opt


def _equal(got, want):
    assert got.keys() == want.keys()
    for name, value in want.items():
        assert got[name].dtype == value.dtype and torch.equal(got[name].float(), value.float()), name


@pytest.mark.parametrize("bits,dtype", [(32, F32), (8, F32), (8, BF16), (32, BF16)])
@pytest.mark.parametrize("in_place", [False, True])
def test_hooks_before_loading_are_followed(bits, dtype, in_place):
    """A hook that matches parameters by their names: the states go where it puts them, in their own types."""
    first, second = _params((20, 30), (20, 30), dtype=dtype)
    saved = _states(AdamW([first, second], state_bits=bits, master=True))
    others = _params((20, 30), (20, 30), dtype=dtype)
    opt = AdamW(others[::-1], state_bits=bits, master=True)

    def match(_, read):
        state = {1 - i: s for i, s in read["state"].items()}
        if in_place:
            read["state"] = state
            return None
        return {**read, "state": state}
    opt.register_load_state_dict_pre_hook(match)
    opt.load_state_dict(saved.state_dict())
    for p, q in zip((first, second), others):
        _equal(opt.state[q], saved.state[p])
    assert not torch.equal(opt.state[others[0]]["exp_avg"].float(), opt.state[others[1]]["exp_avg"].float())
    opt.load_state_dict(saved.state_dict())      # the optimizer's own hooks are gone, the user's stay
    _equal(opt.state[others[0]], saved.state[first])


@pytest.mark.parametrize("prepend", [False, True])
def test_hooks_after_loading_have_the_last_word(prepend):
    """A hook that runs after a load sees the states in their types, and what it changes stays."""
    for bits, dtype in ((32, BF16), (8, BF16), (32, F32)):
        (p,), (q,) = _params((20, 30), dtype=dtype), _params((20, 30), dtype=dtype)
        saved, opt, seen = _states(AdamW([p], state_bits=bits)), AdamW([q], state_bits=bits), []

        def change(opt):
            seen.extend(v.dtype for v in opt.state[q].values())
            opt.state[q]["step"] = torch.tensor(7.0)
            opt.state[q]["exp_avg"].zero_()
        opt.register_load_state_dict_post_hook(change, prepend=prepend)
        opt.load_state_dict(saved.state_dict())
        assert seen == [v.dtype for v in saved.state[p].values()]
        assert float(opt.state[q]["step"]) == 7 and not opt.state[q]["exp_avg"].float().any()
        _equal(opt.state[q], {**saved.state[p], "step": torch.tensor(7.0), "exp_avg": torch.zeros_like(saved.state[p]["exp_avg"].float()).to(
            saved.state[p]["exp_avg"].dtype)})


def _copy(opt):
    """(options of each group, states of each parameter)"""
    return ([{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups],
            [{k: v.clone() for k, v in opt.state[p].items()} for g in opt.param_groups for p in g["params"]])


def _unchanged(opt, before):
    options, states = _copy(opt)
    assert options == before[0] and len(states) == len(before[1])
    for got, want in zip(states, before[1]):
        _equal(got, want)


@pytest.mark.parametrize("name,value", [("lr", -1.0), ("lr", float("nan")), ("betas", (0.9, 1.0)), ("eps", -1.0), ("weight_decay", float("inf")),
                                        ("state_bits", 16), ("seed", 1 << 32)])
def test_a_refused_dict_leaves_the_optimizer_as_it_was(name, value):
    """A number that the constructor refuses, in the last of two groups."""
    groups = lambda: [{"params": [p]} for p in _params((20, 30), (7,))]
    saved = _states(AdamW(groups(), lr=0.25)).state_dict()
    saved["param_groups"][1][name] = value
    opt = _states(AdamW(groups()), seed=5)
    before = _copy(opt)
    with pytest.raises(ValueError):
        opt.load_state_dict(saved)
    _unchanged(opt, before)
    del saved["param_groups"][1]
    with pytest.raises(ValueError):
        opt.load_state_dict(saved)
    _unchanged(opt, before)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("options", [{}, {"foreach": False, "maximize": True}])
def test_a_checkpoint_of_torchs_adamw(dtype, options):
    """States and options of torch's optimizer, which has neither state_bits nor master nor seed."""
    first = _params((20, 30), (7,), (), dtype=dtype)
    theirs = torch.optim.AdamW(first, lr=0.03, betas=(0.8, 0.99), weight_decay=0.2, **options)
    for _ in range(3):
        for p in first:
            p.grad = torch.randn_like(p)
        theirs.step()
    saved = theirs.state_dict()
    opt = AdamW(_params((20, 30), (7,), (), dtype=dtype), lr=1.0, seed=9)
    opt.load_state_dict(saved)
    (group,) = opt.param_groups
    assert (group["lr"], tuple(group["betas"]), group["weight_decay"], group["state_bits"], group["master"], group["seed"]) == (
        0.03, (0.8, 0.99), 0.2, 32, False, 9) and group["maximize"] == options.get("maximize", False)
    for p, q in zip(first, group["params"]):
        got, want = opt.state[q], theirs.state[p]
        assert float(got["step"]) == 3 and got["step"].shape == () and got["step"].dtype == F32
        for name in ("exp_avg", "exp_avg_sq"):
            assert got[name].dtype == F32 and torch.equal(got[name], want[name].float()), name
            assert want[name].dtype == dtype                             # the other optimizer's own
    again = AdamW(_params((20, 30), (7,), (), dtype=dtype))
    again.load_state_dict(opt.state_dict())
    _equal(again.state[again.param_groups[0]["params"][0]], opt.state[group["params"][0]])


def test_a_number_of_steps_that_is_no_tensor():
    saved = _states(AdamW(_params((20, 30)))).state_dict()
    saved["state"][0]["step"] = 11
    opt = AdamW(_params((20, 30)))
    opt.load_state_dict(saved)
    step = opt.state[opt.param_groups[0]["params"][0]]["step"]
    assert float(step) == 11 and step.dtype == F32 and step.shape == ()


@pytest.mark.parametrize("make,bits", [(lambda p: torch.optim.AdamW(p, amsgrad=True), 32), (lambda p: torch.optim.Adam(p, weight_decay=0.1), 32),
                                       (lambda p: torch.optim.AdamW(p), 8)])
def test_checkpoints_of_another_formula_are_refused(make, bits):
    first = _params((20, 30))
    theirs = make(first)
    first[0].grad = torch.ones_like(first[0])
    theirs.step()
    opt = _states(AdamW(_params((20, 30)), state_bits=bits))
    before = _copy(opt)
    with pytest.raises(ValueError):
        opt.load_state_dict(theirs.state_dict())
    _unchanged(opt, before)


_ORDERS = {"rows": lambda p: p, "columns": lambda p: p.transpose(-1, -2).contiguous().transpose(-1, -2),
           "channels last": lambda p: p.contiguous(memory_format=torch.channels_last)}


def _decoded(state, name, p):
    """Moments of 8 bits, laid out as the parameter."""
    axes = sorted(range(p.ndim), key=lambda i: -p.stride(i))
    flat = state[name].float().permute(axes).reshape(-1)
    scales = state[name + "_scale"].repeat_interleave(BLOCK)[:flat.numel()]
    back = sorted(range(p.ndim), key=lambda i: axes[i])
    return (flat * scales).view([p.shape[i] for i in axes]).permute(back)


@pytest.mark.parametrize("shape,orders", [((32, 64), ("rows", "columns")), ((5, 4, 6, 7), ("rows", "channels last"))])
@pytest.mark.parametrize("bits", [8, 32])
def test_another_order_of_memory(shape, orders, bits):
    """States follow their elements into another order; those of 8 bits, whose scales are of the order that was, are refused there."""
    for first in orders:
        for second in orders:
            (p,), (q,) = ([torch.nn.Parameter(_ORDERS[o](t.detach()))] for o, t in zip((first, second), _params(shape) * 2))
            saved, opt = _states(AdamW([p], state_bits=bits)), _states(AdamW([q], state_bits=bits), seed=6)
            before, want = _copy(opt), saved.state[p]
            if bits == 8 and first != second:
                with pytest.raises(CgtpError):
                    opt.load_state_dict(saved.state_dict())
                _unchanged(opt, before)
                continue
            opt.load_state_dict(saved.state_dict())
            assert opt.state[q]["exp_avg"].stride() == q.stride()
            _equal(opt.state[q], want)
            for name in ("exp_avg", "root_avg_sq") if bits == 8 else ():
                assert torch.equal(_decoded(opt.state[q], name, q), _decoded(want, name, p))


def test_one_block_may_change_its_order():
    (p,), (q,) = ([torch.nn.Parameter(_ORDERS[o](t.detach()))] for o, t in zip(("rows", "columns"), _params((16, 16)) * 2))
    saved, opt = _states(AdamW([p], state_bits=8)), AdamW([q], state_bits=8)
    opt.load_state_dict(saved.state_dict())
    assert opt.state[q]["exp_avg"].stride() == (1, 16)
    assert torch.equal(_decoded(opt.state[q], "exp_avg", q), _decoded(saved.state[p], "exp_avg", p))


def test_codes_of_8_bits_are_not_taken_for_numbers():
    """States in 8 bits under an option of 32: left as they are, for the step to refuse."""
    saved = _states(AdamW(_params((20, 30)), state_bits=8)).state_dict()
    saved["param_groups"][0]["state_bits"] = 32
    opt = AdamW(_params((20, 30)))
    opt.load_state_dict(saved)
    assert opt.state[opt.param_groups[0]["params"][0]]["exp_avg"].dtype == E4M3


@pytest.mark.parametrize("bits", [8, 32])
def test_states_are_written_over_where_they_lie(bits):
    """So that what holds their addresses goes on from what was loaded; a dict that shares them, turned round by a hook, too."""
    opt = _states(AdamW(_params((20, 30), (20, 30)), state_bits=bits))
    first, second = opt.param_groups[0]["params"]
    places = [{k: v.data_ptr() for k, v in opt.state[p].items()} for p in (first, second)]
    want = _copy(opt)[1]
    hook = opt.register_load_state_dict_pre_hook(lambda _, read: {**read, "state": {1 - i: s for i, s in read["state"].items()}})
    opt.load_state_dict(opt.state_dict())
    hook.remove()
    for p, s, place in zip((second, first), want, places[::-1]):
        _equal(opt.state[p], s)
        assert {k: v.data_ptr() for k, v in opt.state[p].items()} == place
    saved = _states(AdamW(_params((20, 30), (20, 30)), state_bits=bits), seed=7).state_dict()
    opt.load_state_dict(saved)
    _equal(opt.state[second], saved["state"][1])
    assert {k: v.data_ptr() for k, v in opt.state[second].items()} == places[1]
    opt.state[second]["exp_avg"].copy_(opt.state[first]["exp_avg"])      # the loaded dict's stay as they are
    assert not torch.equal(saved["state"][1]["exp_avg"].float(), opt.state[second]["exp_avg"].float())
