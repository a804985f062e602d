"""What the operators on packed tokens share: argument checks and native calls.

A batch packs the tokens of several scenes in one array; ``scene_starts`` (scenes + 1,)
int32 holds each scene's first row.  The first scene begins at row 0 and the last ends
with the array; entries 0 and ``scenes`` are not read, and the others ascend.  Errors are raised as ValueError
before anything is launched; outputs and workspaces are torch tensors, and
every kernel is enqueued on torch's current stream of the tensors' device.

Calls that the native nodes leave go through autograd functions, also where nothing asks for
a gradient: a trace records them as one operation, whose checks run at each replay, and forward
mode and transforms raise there.
"""
import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from .cuda import _status_error

TYPES = {torch.float32: 0, torch.bfloat16: 1}  # GSV_F32, GSV_BF16
MAX_TOKENS = 2**31 - 2**16  # GSV_MAX_TOKENS

_L = _lib.load()


def call(name, *args):
    st = getattr(_L, "gsv_" + name)(*args)
    if st != 0:
        raise _status_error(name, st)


def stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def workspace_bytes(name, args):
    n = ctypes.c_size_t(0)
    call(name, ctypes.byref(args), ctypes.byref(n))
    return n.value


def check(condition, message):
    if not condition:
        raise ValueError(message)


def activations(t, what, dims, like=None):
    """A float32 or bfloat16 CUDA tensor of `dims` axes, on `like`'s device and of its type."""
    check(isinstance(t, torch.Tensor), f"{what} must be a tensor")
    check(t.is_cuda, f"{what} must be a CUDA tensor")
    check(t.dtype in TYPES, f"{what} must be float32 or bfloat16, got {t.dtype}")
    check(t.dim() == dims, f"{what} must have {dims} axes, got shape {tuple(t.shape)}")
    if like is not None:
        check(t.device == like.device, f"{what} must be on {like.device}, got {t.device}")
        check(t.dtype == like.dtype, f"{what} must be {like.dtype}, got {t.dtype}")
    return t


MAX_ROW_BYTES = 1 << 24


def rows16(t):
    """`t`, or a contiguous copy where its last axis is strided, a row is not 16-byte aligned or
    rows (the third axis from the end) lie more than 16 MB apart.  The stride of an axis of one
    entry says nothing and is not looked at; nor does the C side use it."""
    size = t.element_size()
    strides = [s * size if n > 1 else 0 for s, n in zip(t.stride(), t.shape)]
    if (t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and strides[-3] <= MAX_ROW_BYTES
            and all(s % 16 == 0 for s in strides[:-1])):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def rows(t):
    """`t`, or a contiguous copy where its last axis is strided."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def int32s(t, what, count, device):
    """A contiguous (count,) int32 tensor on `device`."""
    check(isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.dim() == 1,
          f"{what} must be a 1-D int32 tensor")
    check(t.device == device, f"{what} must be on {device}, got {t.device}")
    check(count is None or t.numel() == count, f"{what} must hold {count} values, got {t.numel()}")
    return t.contiguous()


def starts(t, what, device):
    """(the starts, number of scenes) of a packed batch; None is one scene."""
    if t is None:
        return None, 1
    t = int32s(t, what, None, device)
    check(2 <= t.numel() <= MAX_TOKENS, f"{what} must hold scenes + 1 values, got {t.numel()}")
    return t, t.numel() - 1


def fixed(t, what, why):
    """Refuses a tensor that asks for a gradient that the operator does not form (outside the
    autograd functions, whose forward runs without gradients)."""
    check(not (isinstance(t, torch.Tensor) and torch.is_grad_enabled() and t.requires_grad),
          f"{what} get{why} no gradient here: pass {what}.detach()")


def positions(t, what, shape, device):
    """Float32 rows of x, y, z (strided rows, as pos3d_radii[:, :3], are taken as they are)."""
    check(isinstance(t, torch.Tensor) and t.dtype == torch.float32,
          f"{what} must be a float32 tensor")
    check(t.device == device, f"{what} must be on {device}, got {t.device}")
    check(tuple(t.shape) == shape, f"{what} must have shape {shape}, got {tuple(t.shape)}")
    return t if t.stride(-1) == 1 else t.contiguous()


def mask(t, what, shape, device):
    """An int32 (num_tiles_hit serves), bool or uint8 mask: nonzero is kept."""
    check(isinstance(t, torch.Tensor) and t.dtype in (torch.int32, torch.bool, torch.uint8),
          f"{what} must be an int32, bool or uint8 tensor")
    check(t.device == device, f"{what} must be on {device}, got {t.device}")
    check(tuple(t.shape) == shape, f"{what} must have shape {shape}, got {tuple(t.shape)}")
    return t if t.stride(-1) == 1 else t.contiguous()


_ONCE = b"gs_voxelizer: this operator's gradients can be differentiated once only"


def once(backward):
    """A backward whose kernels have no gradients themselves: differentiating its results raises
    (also where the incoming gradient is a constant, so that no second derivative is silently
    left out)."""
    @functools.wraps(backward)
    def wrapped(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():  # no create_graph
            return out
        return tuple(g if g is None else
                     torch._C._functions.DelayedError(_ONCE, 1)(g.detach().requires_grad_())
                     for g in out)
    return wrapped


def present(*tensors):
    """The optional arguments that are given."""
    return [t for t in tensors if t is not None]


def ptr(t):
    return None if t is None else t.data_ptr()


def eager(what):
    """Refuses a call that writes in place where it would be traced or transformed: a trace would hold
    its result and not the call."""
    if (torch._C._get_tracing_state() is not None or torch._C._are_functorch_transforms_active()
            or forward_ad._current_level >= 0):
        raise RuntimeError(f"gs_voxelizer: {what} writes in place and cannot be traced or transformed")


def written(*tensors):
    """Tells autograd that a kernel has written into these tensors."""
    torch.autograd.graph.increment_version([t for t in tensors if t is not None and not t.is_inference()])
