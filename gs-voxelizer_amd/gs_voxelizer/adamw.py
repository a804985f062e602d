"""AdamW over many tensors in one call: the step of a fit of Gaussians, or of a model's training.

    g' = g min(1, max_norm / (|g of all tensors| + 1e-6))       with max_norm, else g
    exp_avg = beta1 exp_avg + (1 - beta1) g'
    exp_avg_sq = beta2 exp_avg_sq + (1 - beta2) g'^2
    w = w (1 - lr weight_decay) - lr / (1 - beta1^t) exp_avg / (sqrt(exp_avg_sq / (1 - beta2^t)) + eps)

`adamw_step` makes one step on given tensors; `AdamW` is the torch optimiser that holds the state.  Parameters
and gradients are float32 or bfloat16, the state is float32, and so is the arithmetic.  A bfloat16
parameter may have a float32 master that the step goes by: the parameter then is its rounded copy, and updates
smaller than its own spacing are not lost.
"""
import ctypes
from typing import Optional, Sequence, Union

import torch
from torch import Tensor

from . import _lib, _native, _tokens as _t


def _each(x, n, what):
    """One value for each tensor."""
    if isinstance(x, (list, tuple)):
        _t.check(len(x) == n, f"{what} must be one value or {n}, got {len(x)}")
        return list(x)
    return [x] * n


def _is_number(x):
    return isinstance(x, (int, float)) and not isinstance(x, bool)


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor],
               exp_avg_sqs: Sequence[Tensor], step: Union[int, Tensor, Sequence[Union[int, Tensor]]], *,
               lr: Union[float, Tensor, Sequence[Union[float, Tensor]]] = 1e-3,
               betas: Sequence[float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: Union[float, Sequence[float]] = 0.0,
               masters: Optional[Sequence[Optional[Tensor]]] = None,
               max_norm: Optional[float] = None) -> Optional[Tensor]:
    """One AdamW step on all tensors, in place.

    Args:
        params: float32 or bfloat16 tensors of one device, without gaps.
        grads: a float32 or bfloat16 gradient each, apart from what the step writes; they are not changed, also
            not by max_norm.
        exp_avgs, exp_avg_sqs: the float32 state, laid out like the params.
        step: the number of this step, from 1, for all tensors or for each; or a (1,) int32 tensor on the
            device that counts the steps made, which the call advances, for all tensors or for each (one that
            several have advances once).  A captured step needs the latter (a number would be the same in
            each replay).
        lr: the rate, or one for each tensor; a number, or a float32 tensor of one element on the device, which a
            captured step reads at each replay.
        weight_decay: of all tensors, or of each.
        masters: for each param a float32 master or None; bfloat16 params only.
        max_norm: the gradients enter as if scaled down so that the norm of all of them is at most this.
    Returns:
        with max_norm the norm of all gradients before that, a float32 tensor; else None.
    """
    if _native.plain():
        done, norm = _native.adamw_step(params, grads, exp_avgs, exp_avg_sqs, masters, step, lr, weight_decay, betas,
                                        eps, max_norm)
        if done:
            return norm
    counter = step if isinstance(step, Tensor) else None
    n = len(params)
    steps = [] if counter is not None else _each(step, n, "step")
    rates, decays = _each(lr, n, "lr"), _each(weight_decay, n, "weight_decay")
    _t.check(max_norm is None or (_is_number(max_norm) and max_norm > 0), f"max_norm must be positive, got {max_norm}")
    for what, values in (("lr", rates), ("weight_decay", decays)):
        for x in values:
            if not (_is_number(x) or (what == "lr" and isinstance(x, Tensor))):
                raise ValueError(f"{what} must be numbers, got {x!r}")
    for x in steps:
        if not isinstance(x, Tensor) and (not isinstance(x, int) or not 1 <= x < 2**53):
            raise ValueError(f"step must be whole numbers from 1, got {x!r}")
    return _step(params, grads, exp_avgs, exp_avg_sqs, masters, steps, counter, rates, decays, betas, eps, max_norm)


def _dense(t):
    """Whether a tensor's elements lie in one run without gaps."""
    if t.is_contiguous():
        return True
    run = 1
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride != run:
            return False
        run *= n
    return True


def _state(t, what, p):
    _t.check(isinstance(t, Tensor) and t.layout == torch.strided and t.dtype == torch.float32
             and t.device == p.device and t.shape == p.shape, f"{what} must be float32, of its param's shape and device")
    _t.check(t.stride() == p.stride() or (t.is_contiguous() and p.is_contiguous()), f"{what} must be laid out like its param")
    return t.data_ptr()


def _step(params, grads, exp_avgs, exp_avg_sqs, masters, steps, counter, rates, decays, betas, eps, max_norm):
    _t.eager("adamw_step")
    n = len(params)
    _t.check(n > 0, "params must hold a tensor")
    for what, ts in (("grads", grads), ("exp_avgs", exp_avgs), ("exp_avg_sqs", exp_avg_sqs), ("masters", masters)):
        _t.check(ts is None or len(ts) == n, f"{what} must hold {n} tensors")
    _t.check(len(betas) == 2 and all(0 <= b < 1 for b in betas), f"betas must be two values from 0 to below 1, got {betas}")
    _t.check(eps >= 0, f"eps must not be negative, got {eps}")
    dev = params[0].device if isinstance(params[0], Tensor) else None
    counters = [counter] if counter is not None else [x for x in steps if isinstance(x, Tensor)]
    for c in counters:
        _t.check(c.dtype == torch.int32 and tuple(c.shape) == (1,) and c.device == dev,
                 f"step must be a number or a (1,) int32 tensor on {dev}")
    held = []  # copies that live until the kernels are enqueued
    entries = (_lib.AdamwTensor * n)()
    for i, (p, g) in enumerate(zip(params, grads)):
        what = f"params[{i}]"
        _t.check(isinstance(p, Tensor) and p.is_cuda and p.layout == torch.strided and p.dtype in _t.TYPES,
                 f"{what} must be a float32 or bfloat16 CUDA tensor")
        _t.check(p.device == dev, f"{what} must be on {dev}, got {p.device}")
        _t.check(_dense(p), f"{what} must not have gaps")
        _t.check(isinstance(g, Tensor) and g.layout == torch.strided and g.dtype in _t.TYPES and g.device == dev
                 and g.shape == p.shape, f"grads[{i}] must be float32 or bfloat16, of its param's shape and device")
        if g.stride() != p.stride():
            g = torch.empty_like(p, dtype=g.dtype).copy_(g.detach())
            held.append(g)
        t = entries[i]
        t.param, t.grad, t.numel = p.data_ptr(), g.data_ptr(), p.numel()
        t.exp_avg = _state(exp_avgs[i], f"exp_avgs[{i}]", p)
        t.exp_avg_sq = _state(exp_avg_sqs[i], f"exp_avg_sqs[{i}]", p)
        if masters is not None and masters[i] is not None:
            _t.check(p.dtype == torch.bfloat16, f"masters[{i}]: {what} is float32 and needs none")
            t.master = _state(masters[i], f"masters[{i}]", p)
        rate, decay = rates[i], decays[i]
        if isinstance(rate, Tensor):
            _t.check(rate.dtype == torch.float32 and rate.numel() == 1 and rate.device == dev,
                     f"lr must be numbers or float32 tensors of one element on {dev}")
            t.lr_device = rate.data_ptr()
        else:
            _t.check(rate >= 0, f"lr must not be negative, got {rate}")
            t.lr = rate
        _t.check(decay >= 0, f"weight_decay must not be negative, got {decay}")
        t.weight_decay = decay
        if counter is None and isinstance(steps[i], Tensor):
            t.counter = steps[i].data_ptr()
        elif counter is None:
            t.step = steps[i]
        t.dtype, t.grad_dtype = _t.TYPES[p.dtype], _t.TYPES[g.dtype]
    a = _lib.Adamw(tensors=ctypes.addressof(entries), count=n, beta1=betas[0], beta2=betas[1], eps=eps,
                   max_norm=max_norm or 0.0, counter=_t.ptr(counter))
    norm = None
    with torch.cuda.device(dev):
        if counter is None and len(counters) < n and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("gs_voxelizer: a captured step needs its count on the device (a (1,) int32 tensor)")
        if max_norm:
            norm = torch.empty((), dtype=torch.float32, device=dev)
            a.norm = norm.data_ptr()
        size = _t.workspace_bytes("adamw_workspace_bytes", a)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        try:
            _t.call("adamw", ctypes.byref(a), ws.data_ptr(), size, _t.stream(dev))
        except RuntimeError as e:
            # (what else the library refuses is checked above)
            if "argument" not in str(e):
                raise
            raise ValueError(f"{e}: a tensor that the step writes shares memory with another, or with a gradient")
    _t.written(*params, *exp_avgs, *exp_avg_sqs, *(masters or []), *counters)
    return norm


class AdamW(torch.optim.Optimizer):
    """AdamW whose step is `adamw_step`: one call for all parameters, whatever their groups' rates and
    decays are.

    Args:
        params: parameters or groups of them, with ``lr``, ``betas``, ``eps`` and ``weight_decay`` each.
        masters: bfloat16 parameters get float32 masters (state ``master``), which the steps go by.
        max_norm: see `adamw_step`; over all groups, which then have one device, ``betas`` and ``eps``.  The last
            step's norm is ``self.norm``.
        capturable: (likewise one device, ``betas`` and ``eps``) each parameter's steps are counted on the device, and
            the step can be captured in a graph once an ordinary step has been made with the same gradients
            there.  ``lr`` may be a float32 tensor of one element on the device.

    Each parameter counts the steps that it made itself: one without a gradient at some step is left as it is and
    does not count it.

    A step that is captured together with a voxelization would be made twice where
    `graph.CapturedStep` has to run a replay again: capture the optimiser's step in a graph of its own.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, masters: bool = False,
                 max_norm: Optional[float] = None, capturable: bool = False):
        _t.check(isinstance(lr, Tensor) or lr >= 0, f"lr must not be negative, got {lr}")
        _t.check(len(betas) == 2 and all(0 <= b < 1 for b in betas),
                 f"betas must be two values from 0 to below 1, got {betas}")
        _t.check(eps >= 0, f"eps must not be negative, got {eps}")
        _t.check(weight_decay >= 0, f"weight_decay must not be negative, got {weight_decay}")
        _t.check(max_norm is None or max_norm > 0, f"max_norm must be positive, got {max_norm}")
        self.masters, self.max_norm, self.capturable = masters, max_norm, capturable
        self.norm: Optional[Tensor] = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def _new_state(self, p):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("gs_voxelizer: the first step makes the optimiser's state: run one before the capture")
        s = self.state[p]
        s["step"] = torch.zeros(1, dtype=torch.int32, device=p.device) if self.capturable else 0
        s["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        s["exp_avg_sq"] = torch.zeros_like(s["exp_avg"])
        if self.masters and p.dtype == torch.bfloat16:
            s["master"] = p.detach().to(torch.float32)
        return s

    @torch.no_grad()
    def step(self, closure=None):
        """One step; returns the closure's loss, if there is one."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        calls = {}
        for group in self.param_groups:
            key = (tuple(group["betas"]), group["eps"])
            for p in group["params"]:
                if p.grad is None:
                    continue
                s = self.state.get(p) or self._new_state(p)
                calls.setdefault((p.device, *key), []).append((p, s, group["lr"], group["weight_decay"]))
        _t.check((self.max_norm is None and not self.capturable) or len(calls) <= 1,
                 "max_norm and capturable need parameters of one device, and one betas and eps in all groups")
        for (_, betas, eps), members in calls.items():
            ps, states = [c[0] for c in members], [c[1] for c in members]
            count = [s["step"] if self.capturable else s["step"] + 1 for s in states]
            self.norm = adamw_step(
                ps, [p.grad for p in ps], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], count,
                lr=[c[2] for c in members], betas=betas, eps=eps, weight_decay=[c[3] for c in members],
                masters=[s.get("master") for s in states] if self.masters else None, max_norm=self.max_norm)
            if not self.capturable:
                for s in states:
                    s["step"] += 1
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, but the state is float32 whatever the parameters' type is, and copied.  A saved master is taken
        where this optimiser keeps one for the parameter; where none was saved the parameter's value becomes it (so load
        the model's weights first).
        Raises ValueError, and loads nothing, where the state is another optimiser's or of other shapes.  A graph
        captured before steps the state that there was: capture again."""
        saved = state_dict["state"]
        for g in state_dict["param_groups"]:
            _t.check(not (g.get("maximize") or g.get("amsgrad"))
                     and (g.get("decoupled_weight_decay", True) or not g.get("weight_decay")),
                     "the state of an optimiser that maximizes, has amsgrad or adds the decay to the gradients")
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            for name in ("step", "exp_avg", "exp_avg_sq", "master") if saved.get(i) else ():
                _t.check(name in saved[i] or name == "master", f"the state of parameter {i} has no {name}")
                _t.check(name == "step" or name not in saved[i] or saved[i][name].shape == p.shape,
                         f"{name} of parameter {i} must have shape {tuple(p.shape)}")
        super().load_state_dict(state_dict)
        for i, p in zip(ids, params):
            if not saved.get(i):  # (empty where a state was looked at that there was none of)
                continue
            s = self.state[p] = {}
            mastered = self.masters and p.dtype == torch.bfloat16
            for name, x in saved[i].items():
                if name == "master" and not mastered:
                    continue  # no step would keep it up to date
                s[name] = (int(x) if name == "step" else
                           torch.empty_like(p, dtype=torch.float32).copy_(x) if isinstance(x, Tensor) else x)
            if mastered and "master" not in s:
                s["master"] = p.detach().to(torch.float32)
            if self.capturable:
                s["step"] = torch.tensor([s["step"]], dtype=torch.int32, device=p.device)

    def __getstate__(self):
        return {**super().__getstate__(), "masters": self.masters, "max_norm": self.max_norm,
                "capturable": self.capturable, "norm": self.norm}
