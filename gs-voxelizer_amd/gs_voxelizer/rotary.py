"""Rotary positions with several axes, for tokens that lie in a volume.

The angle of channel pair p at token t is ``theta[t, p] = sum_a positions[t, a] *
frequencies[a, p]``: with one nonzero frequency a pair (`axis_frequencies`) each pair turns
with one axis, with several it turns along a direction.  A pair (x1, x2) becomes
(x1 cos - x2 sin, x1 sin + x2 cos); the gradient is the rotation back.  float32 and
bfloat16, angles formed in binary64; no gradient for positions and frequencies.
"""
import ctypes
from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor
from torch.autograd import Function

from . import _lib, _native, _tokens as _t


def axis_frequencies(pairs: Sequence[int], base: float = 1000.0, device=None) -> Tensor:
    """(axes, sum(pairs)) frequencies: the first pairs[0] channel pairs turn with axis 0,
    the next pairs[1] with axis 1, and so on, geometrically from 1 to about 1 / base."""
    _t.check(len(pairs) > 0 and all(int(n) >= 0 for n in pairs) and sum(pairs) > 0,
             f"pairs must be counts for each axis, got {pairs}")
    _t.check(base > 0, f"base must be positive, got {base}")
    f = torch.zeros(len(pairs), sum(pairs), dtype=torch.float32)
    first = 0
    for a, n in enumerate(pairs):
        f[a, first:first + n] = base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))
        first += n
    return f.to(device)


def rotate_qk(q: Tensor, k: Optional[Tensor], positions: Tensor, frequencies: Tensor,
              interleaved: bool = False) -> Tuple[Tensor, Optional[Tensor]]:
    """Turn the heads of q (T, H, D) and k (T, K, D) by their tokens' positions.

    Args:
        q, k: float32 or bfloat16, the last axis contiguous (views into one projection's
            output are taken as they are); k may be None.
        positions: (T, A) float32, e.g. the centres pos3d_radii[:, :3] in voxel units.
        frequencies: (A, P) float32 with 2 P <= D.
        interleaved: pair p is channels (2p, 2p + 1) instead of (p, P + p).
    Returns:
        the turned q and k, contiguous; channels from 2 P on pass through.
    """
    if k is not None and _native.plain(q, k, positions, frequencies):
        out = _native.rotate(q, k, positions, frequencies, bool(interleaved))
        if out:
            return tuple(out)
    _t.fixed(positions, "positions", "")
    _t.fixed(frequencies, "frequencies", "")
    return _RotateQK.apply(q, k, positions, frequencies, bool(interleaved))


def _checked(q, k, positions, frequencies):
    """The frequencies as the kernel takes them."""
    _t.activations(q, "q", 3)
    dev = q.device
    if k is not None:
        _t.activations(k, "k", 3, like=q)
        _t.check(k.shape[0] == q.shape[0] and k.shape[2] == q.shape[2],
                 f"k must have q's tokens and channels, got {tuple(k.shape)} for {tuple(q.shape)}")
    T, _, D = q.shape
    for t, what in ((positions, "positions"), (frequencies, "frequencies")):
        _t.check(isinstance(t, Tensor) and t.dtype == torch.float32 and t.dim() == 2,
                 f"{what} must be a 2-D float32 tensor")
        _t.check(t.device == dev, f"{what} must be on {dev}, got {t.device}")
    A, P = frequencies.shape
    _t.check(tuple(positions.shape) == (T, A),
             f"positions must have shape {(T, A)}, got {tuple(positions.shape)}")
    _t.check(1 <= A <= 8, f"frequencies must have 1 to 8 axes, got {A}")
    _t.check(P >= 1 and 2 * P <= D, f"{P} channel pairs do not fit {D} channels")
    _t.check(D <= 1024, f"at most 1024 channels, got {D}")
    _t.check(q.shape[1] + (0 if k is None else k.shape[1]) <= 4096, "at most 4096 heads")
    _t.check(T <= _t.MAX_TOKENS, "too many tokens")
    return frequencies.contiguous()


def _turn(q, k, positions, frequencies, interleaved, inverse):
    """The native call; q or k may be None."""
    one = q if q is not None else k
    q_out = k_out = None
    a = _lib.Rotary(positions=positions.data_ptr(), frequencies=frequencies.data_ptr(),
                    pos_row=positions.stride(0), pos_axis=positions.stride(1),
                    dtype=_t.TYPES[one.dtype], tokens=one.shape[0], dim=one.shape[2],
                    pairs=frequencies.shape[1], axes=frequencies.shape[0], interleaved=interleaved)
    if q is not None:
        q = _t.rows(q)
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        a.q, a.q_row, a.q_head, a.heads = q.data_ptr(), q.stride(0), q.stride(1), q.shape[1]
    if k is not None:
        k = _t.rows(k)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        a.k, a.k_row, a.k_head, a.kv_heads = k.data_ptr(), k.stride(0), k.stride(1), k.shape[1]
    if one.numel():
        with torch.cuda.device(one.device):
            _t.call("rotary", ctypes.byref(a), _t.ptr(q_out), _t.ptr(k_out), int(inverse),
                    _t.stream(one.device))
    return q_out, k_out


class _RotateQK(Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequencies, interleaved):
        frequencies = _checked(q, k, positions, frequencies)
        ctx.interleaved = interleaved
        ctx.save_for_backward(positions, frequencies)
        ctx.set_materialize_grads(False)
        return _turn(q, k, positions, frequencies, interleaved, False)

    @staticmethod
    @_t.once
    def backward(ctx, dq, dk):
        dq, dk = (g if need else None for g, need in zip((dq, dk), ctx.needs_input_grad))
        if dq is None and dk is None:
            return None, None, None, None, None
        positions, frequencies = ctx.saved_tensors
        dq, dk = _turn(dq, dk, positions, frequencies, ctx.interleaved, True)
        return dq, dk, None, None, None
