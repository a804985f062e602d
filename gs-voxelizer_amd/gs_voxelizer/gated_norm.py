"""The norms around a block of a token model, fused with its gate and residual scale.

    n = branch * rstd(branch) * branch_weight     (or n = branch)
    y = x + gate * scale * n                      h = y * rstd(y) * weight

with rstd(v) = 1 / sqrt(mean(v^2) + eps) over a row: what a residual block does with
its branch's output and what the next block reads.  One pass over the rows each way, sums
and norms in float32, deterministic parameter gradients.
"""
import ctypes
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import Function

from . import _lib, _native, _tokens as _t

MAX_CHANNELS = 8192


def gated_residual_norm(x: Tensor, branch: Tensor, weight: Tensor, *,
                        branch_weight: Optional[Tensor] = None, scale: Optional[Tensor] = None,
                        gate: Optional[Tensor] = None, scene_starts: Optional[Tensor] = None,
                        longest: Optional[int] = None, eps: float = 1e-6) -> Tuple[Tensor, Tensor]:
    """Add a block's output to the residual stream and norm the sum.

    Args:
        x: (T, C) residual stream, float32 or bfloat16.
        branch: (T, C) the block's output: x's type, or bfloat16 beside a float32 x.
        weight: (C,) float32, of the norm after the sum.
        branch_weight: (C,) float32: the branch is normed first; None: it is not.
        scale: (C,) float32 residual scale, or None.
        gate: a row for each scene (scenes, C) with scene_starts, for each token (T, C), or
            (1, C) for all of them; float32 or branch's type; or None.
        scene_starts: (scenes + 1,) int32 first rows of the scenes.
        longest: rows of the longest scene, taken so that one packing's arguments serve all
            operators; nothing here depends on it.
    Returns:
        y (T, C) of x's type and h (T, C) of branch's type.
    """
    if _native.plain(x, branch, weight, *_t.present(branch_weight, scale, gate, scene_starts)):
        out = _native.gated_norm(x, branch, weight, branch_weight, scale, gate, scene_starts,
                                 float(eps))
        if out:
            return tuple(out)
    return _GatedNorm.apply(x, branch, weight, branch_weight, scale, gate, scene_starts, eps)


def _checked(x, branch, weight, branch_weight, scale, gate, scene_starts, eps):
    """The starts that matter, and what else _args takes."""
    _t.activations(x, "x", 2)
    _t.activations(branch, "branch", 2)
    dev, (T, C) = x.device, x.shape
    _t.check(branch.shape == x.shape and branch.device == dev,
             f"branch must have x's shape {tuple(x.shape)} and device")
    _t.check(branch.dtype == x.dtype or x.dtype == torch.float32,
             f"branch must be bfloat16 where x is, got {branch.dtype}")
    _t.check(1 <= C <= MAX_CHANNELS, f"1 to {MAX_CHANNELS} channels, got {C}")
    _t.check(T <= _t.MAX_TOKENS, "too many tokens")
    for t, what in ((weight, "weight"), (branch_weight, "branch_weight"), (scale, "scale")):
        if t is None and what != "weight":
            continue
        _t.check(isinstance(t, Tensor) and t.dtype == torch.float32 and tuple(t.shape) == (C,)
                 and t.device == dev, f"{what} must be a ({C},) float32 tensor on {dev}")
    starts, scenes = _t.starts(scene_starts, "scene_starts", dev)
    per_token = False
    if gate is not None:
        _t.activations(gate, "gate", 2)
        _t.check(gate.device == dev and gate.dtype in (torch.float32, branch.dtype),
                 f"gate must be float32 or {branch.dtype}, on {dev}")
        per_token = starts is None and gate.shape[0] == T and T != 1
        _t.check(gate.shape[1] == C and (per_token or gate.shape[0] == scenes),
                 f"gate must have a row for each of {scenes} scene(s)"
                 + ("" if starts is not None else f" or {T} tokens")
                 + f" and {C} channels, got {tuple(gate.shape)}")
    _t.check(eps >= 0, f"eps must not be negative, got {eps}")
    if gate is None or per_token:
        starts, scenes = None, 1  # no value depends on the scenes
    return starts, (per_token, scenes, float(eps))


def _args(x, branch, weight, branch_weight, scale, gate, starts, opts):
    """The native call's arguments, and the tensors they point into."""
    per_token, scenes, eps = opts
    x, branch = _t.rows(x), _t.rows(branch)
    held = [x, branch] + [t if t is None else t.contiguous() for t in (weight, branch_weight, scale)]
    if gate is not None:
        gate = _t.rows(gate)
    a = _lib.Norm(x=x.data_ptr(), branch=branch.data_ptr(), weight=held[2].data_ptr(),
                  branch_weight=_t.ptr(held[3]), scale=_t.ptr(held[4]), starts=_t.ptr(starts),
                  x_row=x.stride(0), branch_row=branch.stride(0), dtype=_t.TYPES[x.dtype],
                  branch_dtype=_t.TYPES[branch.dtype], tokens=x.shape[0], channels=x.shape[1],
                  scenes=scenes, eps=eps)
    if gate is not None:
        a.gate, a.gate_row, a.gate_dtype = gate.data_ptr(), gate.stride(0), _t.TYPES[gate.dtype]
        a.gate_per_token = per_token
    return a, held + [gate]


def _forward(x, branch, weight, branch_weight, scale, gate, starts, opts):
    a, held = _args(x, branch, weight, branch_weight, scale, gate, starts, opts)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = torch.empty(x.shape, dtype=branch.dtype, device=x.device)
    if x.shape[0]:
        with torch.cuda.device(x.device):
            _t.call("gated_norm_fwd", ctypes.byref(a), y.data_ptr(), h.data_ptr(),
                    _t.stream(x.device))
    return y, h


class _GatedNorm(Function):
    @staticmethod
    def forward(ctx, x, branch, weight, branch_weight, scale, gate, scene_starts, eps):
        starts, ctx.opts = _checked(x, branch, weight, branch_weight, scale, gate, scene_starts, eps)
        ctx.save_for_backward(x, branch, weight, branch_weight, scale, gate, starts)
        ctx.set_materialize_grads(False)
        return _forward(x, branch, weight, branch_weight, scale, gate, starts, ctx.opts)

    @staticmethod
    @_t.once
    def backward(ctx, dy, dh):
        x, branch, weight, branch_weight, scale, gate, starts = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 8
        a, held = _args(x, branch, weight, branch_weight, scale, gate, starts, ctx.opts)
        dev = x.device
        dy, dh = (t if t is None else _t.rows(t) for t in (dy, dh))
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
        dbranch = torch.empty(x.shape, dtype=branch.dtype, device=dev)
        dw, dbw, ds = (None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)
                       for t in (weight, branch_weight, scale))
        dg = None if gate is None else torch.empty(gate.shape, dtype=gate.dtype, device=dev)
        with torch.cuda.device(dev):
            n = _t.workspace_bytes("gated_norm_bwd_workspace_bytes", a)
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
            _t.call("gated_norm_bwd", ctypes.byref(a), _t.ptr(dy), 0 if dy is None else dy.stride(0),
                    _t.ptr(dh), 0 if dh is None else dh.stride(0), dx.data_ptr(),
                    dbranch.data_ptr(), dw.data_ptr(), _t.ptr(dbw), _t.ptr(ds), _t.ptr(dg),
                    ws.data_ptr(), n, _t.stream(dev))
        return dx, dbranch, dw, dbw, ds, dg, None, None
