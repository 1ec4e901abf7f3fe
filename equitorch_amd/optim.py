"""AdamW over all tensors of a model at once, with states in 32 bits or in 8.

``cgtp_adamw_step`` takes dozens of tensors a launch.  The step's numbers are on the GPU, so that a recorded graph that holds a
step counts on when it is replayed."""
import ctypes as C
from typing import Iterable, Optional, Tuple, Union

import torch
from torch import Tensor

from . import _lib, _shim
from ._lib import AdamwArgs, AdamwTensor, CgtpError

BLOCK = 256        # elements that share a scale
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_E4M3 = torch.float8_e4m3fn
_OPTIONS = ("lr", "betas", "eps", "weight_decay", "state_bits", "master", "maximize", "seed")


def _dense(t: Tensor) -> bool:
    """Whether the elements lie one after the other, in any order of the axes."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _same_order(a: Tensor, b: Tensor) -> bool:
    """Whether the elements of two tensors of one shape lie in the same order (the stride of an axis of one says nothing)."""
    return all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def _like(p: Tensor, dtype: torch.dtype) -> Tensor:
    """Zeros in the order of p's elements."""
    if dtype == _E4M3:
        return torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.preserve_format).view(_E4M3)
    return torch.zeros_like(p, dtype=dtype, memory_format=torch.preserve_format)


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay (``torch.optim.AdamW``'s formula) for fp32, bf16 and fp16 parameters on the GPU.

    ``state_bits``: 32, ``exp_avg`` and ``exp_avg_sq`` in fp32; or 8, ``exp_avg`` and ``root_avg_sq`` (its square root) in
    ``torch.float8_e4m3fn``, each with a ``..._scale`` in fp32 for every 256 elements in the order of memory.  ``root_avg_sq`` is rounded up or
    down at random in proportion, since a step's change of it is far below the distance of two such values; the random bits are
    a hash of ``seed``, the parameter's place among all of the optimizer's, the step and the element, so runs repeat.  A block of 256
    with a gradient that is not finite, or whose square is not, becomes NaN.

    ``master``: parameters in 16 bits have a copy in fp32 (``master``) that the steps are taken on, and receive it rounded.  Without it
    a step below half a unit of a 16-bit weight is lost.  Weights that are written into such a parameter from elsewhere have to be written into the copy
    too: the next step is taken on that.

    ``lr`` may be an fp32 tensor on the GPU, which is read when the step runs: a recorded graph then follows it.  Every number else
    is fixed when a graph records the step, and states have to be there by then (one step before).  ``step`` in a parameter's state counts on the
    GPU.  Parameters without a gradient are passed over."""

    _made = True                                 # whether the groups are there: a copy's, whose constructor does not run

    def __init__(self, params: Iterable, lr: Union[float, Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, master: bool = False, maximize: bool = False, seed: int = 0):
        self._made = False
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, master=master,
                                      maximize=maximize, seed=seed))
        self._made = True
        self._check_overlap()                    # once for all groups

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        try:
            self._check_numbers(self.param_groups[-1])
            if self._made:
                self._check_overlap()
        except ValueError:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_numbers(group: dict) -> None:
        lr = group["lr"]
        if isinstance(lr, Tensor):
            if lr.numel() != 1 or (lr.is_cuda and lr.dtype != torch.float32):
                raise ValueError(f"lr must be a number or one fp32 number on the GPU, got {lr.dtype} {tuple(lr.shape)}")
            lr = None if lr.is_cuda else lr.item()      # on the GPU it is read when the kernels run
        if lr is not None and not 0.0 <= lr < float("inf"):
            raise ValueError(f"lr must be finite and not negative, got {lr}")
        betas = group["betas"]
        if len(betas) != 2 or not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas must be two numbers of 0 <= beta < 1, got {betas}")
        if not 0.0 <= group["weight_decay"] < float("inf"):
            raise ValueError(f"weight_decay must be finite and not negative, got {group['weight_decay']}")
        if not (group["eps"] == 0.0 or 2.0 ** -126 <= group["eps"] <= 2.0 ** 128 * (1 - 2.0 ** -24)):
            raise ValueError(f"eps must be 0, or above it in fp32's range, got {group['eps']}")
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {group['state_bits']}")
        if not 0 <= group["seed"] < 1 << 32:
            raise ValueError(f"seed must be 0 <= seed < 2^32, got {group['seed']}")

    def _check_overlap(self) -> None:
        taken = []
        for p in (p for g in self.param_groups for p in g["params"]):
            if p.numel():
                last = sum((n - 1) * s for n, s in zip(p.shape, p.stride()))
                taken.append((str(p.device), p.data_ptr(), p.data_ptr() + (last + 1) * p.element_size()))
        taken.sort()
        for (d, _, end), (e, begin, _) in zip(taken, taken[1:]):
            if d == e and d != "meta" and begin < end:
                raise ValueError("parameters overlap in memory, or one is given twice: a step would update the same elements twice")

    def load_state_dict(self, state_dict: dict) -> None:
        """As torch's, hooks included, with every state in its own type (torch's takes floating-point states to the parameter's).  A dict of
        ``torch.optim.AdamW`` is taken too: options that it does not have keep their values, ``exp_avg`` and ``exp_avg_sq`` become fp32.  What
        is refused leaves the optimizer as it was.

        States that are there, and an ``lr`` on the GPU (unless groups that share it come with several), are written over where they lie: a
        recorded graph that holds a step goes on from what was loaded."""
        loaded = []

        def check(_, read):
            read = self._completed(read)
            loaded.extend((read, {p: dict(s) for p, s in self.state.items()}, [g["lr"] for g in self.param_groups]))
            return read
        # last of the hooks before, first of those after: the states are those of the dict that the others leave, and stay what the others make of them
        handles = [self.register_load_state_dict_pre_hook(check),
                   self.register_load_state_dict_post_hook(lambda _: self._load_states(*loaded), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for handle in handles:
                handle.remove()

    def _completed(self, state_dict: dict) -> dict:
        """The dict with options and states as a step takes them."""
        saved = state_dict["param_groups"]
        if [len(g["params"]) for g in saved] != [len(g["params"]) for g in self.param_groups]:
            return state_dict                    # torch refuses it
        groups = [{**{k: now[k] for k in _OPTIONS}, **g} for now, g in zip(self.param_groups, saved)]
        state = dict(state_dict["state"])
        for now, group in zip(self.param_groups, groups):
            self._check_numbers(group)
            if group.get("amsgrad") or (group["weight_decay"] and not group.get("decoupled_weight_decay", True)):
                raise ValueError("the dict is of another formula: amsgrad, or a weight decay that is added to the gradient")
            for p, i in zip(now["params"], group["params"]):
                if not state.get(i):
                    continue
                s = state[i] = dict(state[i])
                if group["state_bits"] == 8 and "exp_avg_sq" in s:
                    raise ValueError("states in 32 bits do not fit state_bits = 8: load them into an optimizer of 32")
                for name in ("exp_avg", "root_avg_sq") if group["state_bits"] == 8 else ():
                    t = s.get(name)
                    # the scales are those of 256 elements each in the order of memory as it was: of one block alone in any order
                    if isinstance(t, Tensor) and t.shape == p.shape and p.numel() > BLOCK and not _same_order(t, p):
                        raise CgtpError(f"state {name!r} in 8 bits was saved in another order of memory (strides {t.stride()}) than that of its parameter "
                                        f"(strides {p.stride()} of {tuple(p.shape)}), whose blocks its scales do not fit")
                if "step" in s:
                    s["step"] = torch.as_tensor(s["step"], dtype=torch.float32).reshape(())
                for name in ("exp_avg", "exp_avg_sq") if group["state_bits"] == 32 else ():
                    if isinstance(s.get(name), Tensor) and s[name].dtype in (torch.bfloat16, torch.float16, torch.float64):
                        s[name] = s[name].float()
        return {**state_dict, "state": state, "param_groups": groups}

    @torch.no_grad()
    def _load_states(self, state_dict: dict, before: dict, rates: list) -> None:
        """before, rates: the states and learning rates that the load replaced."""
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        there = {t.untyped_storage().data_ptr() for s in before.values() for t in s.values() if isinstance(t, Tensor)}
        values = []
        for i, p in zip(ids, params):
            for name, value in state_dict["state"].get(i, {}).items():
                if isinstance(value, Tensor):        # a state that the dict shares with this optimizer may be written over before its turn
                    values.append((p, name, value.clone() if value.untyped_storage().data_ptr() in there else value))
        for p, name, value in values:
            like_p, old = value.shape == p.shape and value.ndim, before.get(p, {}).get(name)
            if isinstance(old, Tensor) and (old.shape, old.dtype, old.device) == (value.shape, value.dtype, p.device) and (
                    _same_order(old, p) if like_p else old.is_contiguous()):
                old.copy_(value)
            elif like_p:
                old = _like(p, value.dtype).copy_(value)
            else:
                old = value.to(p.device, copy=True)
            self.state[p][name] = old
        for lr in {id(t): t for t in rates if isinstance(t, Tensor) and t.is_cuda}.values():
            sharing = [g for g, t in zip(self.param_groups, rates) if t is lr]
            if len({float(g["lr"]) for g in sharing}) == 1:      # else each group has its own from now on
                lr.fill_(float(sharing[0]["lr"]))
                for group in sharing:
                    group["lr"] = lr

    def _init_state(self, p: Tensor, bits: int, master: bool) -> dict:
        if torch.cuda.is_current_stream_capturing():
            raise CgtpError("states would be made anew by every replay: take one step before a graph records one")
        state = self.state[p]
        state["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
        if bits == 32:
            state["exp_avg"], state["exp_avg_sq"] = _like(p, torch.float32), _like(p, torch.float32)
        else:
            for name in ("exp_avg", "root_avg_sq"):
                state[name] = _like(p, _E4M3)
                state[name + "_scale"] = torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)
        if master and p.dtype != torch.float32:
            state["master"] = _like(p, torch.float32).copy_(p)
        return state

    def _operands(self, p: Tensor, bits: int, master: bool):
        """(grad, exp_avg, exp_avg_sq, their scales, master, step) as the kernels take them."""
        g = p.grad
        if g.layout != torch.strided:
            raise CgtpError(f"gradients must be dense, got {g.layout}")
        if not p.is_cuda or p.dtype not in _DTYPES:
            raise CgtpError(f"parameters must be fp32, bf16 or fp16 on the GPU, got {p.dtype} on {p.device}")
        if g.dtype != p.dtype or g.device != p.device or g.shape != p.shape:
            raise CgtpError(f"a gradient must be of its parameter's type, device and shape, got {g.dtype} {tuple(g.shape)} on {g.device}")
        if not _dense(p):
            raise CgtpError(f"a parameter's elements must lie one after the other, got strides {p.stride()} of {tuple(p.shape)}")
        if p.numel() >= 1 << 31:
            raise CgtpError(f"a parameter must have fewer than 2^31 elements, got {p.numel()}")
        if not _same_order(g, p):
            g = torch.empty_like(p).copy_(g)
        state = self.state[p] or self._init_state(p, bits, master)
        wide, blocks = (torch.float32, _E4M3)[bits == 8], (-(-p.numel() // BLOCK),)
        names = ("exp_avg", "exp_avg_sq") if bits == 32 else ("exp_avg", "root_avg_sq")
        wanted = [(n, wide, p.shape) for n in names]
        wanted += [(n + "_scale", torch.float32, blocks) for n in names] if bits == 8 else []
        wanted += [("master", torch.float32, p.shape)] if master and p.dtype != torch.float32 else []
        for name, dtype, shape in wanted + [("step", torch.float32, ())]:
            t = state.get(name)
            if not isinstance(t, Tensor) or t.dtype != dtype or t.shape != shape or t.device != p.device \
                    or not (_same_order(t, p) if shape == p.shape else t.is_contiguous()):
                raise CgtpError(f"state {name!r} of a parameter {tuple(p.shape)} must be {dtype} {tuple(shape)} on {p.device}, in the order "
                                f"of the parameter's elements: it is missing or another (state_bits or master of another run?)")
        scales = [state[n + "_scale"] for n in names] if bits == 8 else [None, None]
        return g, *[state[n] for n in names], *scales, state["master"] if master and p.dtype != torch.float32 else None, state["step"]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:          # a schedule or a user may have changed them; nothing is stepped if one is refused
            self._check_numbers(group)
        mod, number = _shim.module(), 0
        for group in self.param_groups:
            params, lr, (b1, b2) = group["params"], group["lr"], group["betas"]
            on_gpu = isinstance(lr, Tensor) and lr.is_cuda
            a = AdamwArgs()
            a.lr, a.beta1, a.beta2, a.eps, a.weight_decay = 0.0 if on_gpu else float(lr), b1, b2, group["eps"], group["weight_decay"]
            a.lr_ptr = lr.data_ptr() if on_gpu else None
            a.state_bits, a.maximize, a.seed = group["state_bits"], group["maximize"], group["seed"]
            if mod is None or not mod.adamw(params, self.state, group["master"], lr if on_gpu else None, C.addressof(a), number):
                self._step_group(params, a, group["master"], number, lr if on_gpu else None)
            number += len(params)
        return loss

    def _step_group(self, params, a: AdamwArgs, master: bool, number: int, lr: Optional[Tensor]) -> None:
        """One call for each device and type: what the extension does where every operand is as the kernels take it."""
        calls = {}
        for i, p in enumerate(params):
            if p.grad is not None:
                calls.setdefault((p.device, p.dtype), []).append((i, p, self._operands(p, a.state_bits, master)))
        for device, _ in calls:
            if lr is not None and lr.device != device:
                raise CgtpError(f"lr is on {lr.device}, parameters on {device}")
        for (device, dtype), items in calls.items():
            tensors = (AdamwTensor * len(items))()
            for t, (i, p, (g, m, v, m_scale, v_scale, wide, step)) in zip(tensors, items):
                t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.step = (x.data_ptr() for x in (p, g, m, v, step))
                t.exp_avg_scale, t.exp_avg_sq_scale, t.master = _lib.ptr(m_scale), _lib.ptr(v_scale), _lib.ptr(wide)
                t.n, t.number = p.numel(), number + i
            a.tensors, a.n_tensors, a.dtype = tensors, len(items), _lib.dtype_code(dtype)
            a.master = int(master and dtype != torch.float32)
            with torch.cuda.device(device):
                _lib.check(_lib.lib.cgtp_adamw_step(C.byref(a), _lib.stream_ptr(device)), "cgtp_adamw_step")
            torch.autograd.graph.increment_version([p for _, p, _ in items])
