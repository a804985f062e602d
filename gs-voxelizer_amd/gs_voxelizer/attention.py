"""Attention among the tokens of packed scenes, and of new tokens over a cache.

    t_ij = scale q_i.k_j                   capped: cap tanh(scale q_i.k_j / cap)
    t_ij -= slopes[h] |p_i - p_j|          with a distance bias
    out_i = sum_j softmax_j(t_ij) v_j      0 for a token that sees no key

A token sees the kept keys of its own scene; with ``causal`` those up to itself and the
scene's prefix.  float32 and bfloat16; scores, softmax and sums in float32.  Gradients for q,
k, v and slopes run in a fixed order (the same inputs give the same bits); positions get
none.  A NaN or infinity in a key that is masked out by scene, keep or length reaches
nothing; one in a key that only causality hides from some tokens can reach those in the same
tile.
"""
import ctypes
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import Function

from . import _lib, _native, _tokens as _t

MAX_DIM = 128


def _heads(q, k, v, dims):
    _t.activations(q, "q", 3)
    _t.activations(k, "k", dims, like=q)
    _t.activations(v, "v", dims, like=q)
    _t.check(k.shape == v.shape, f"k and v must have one shape, got {tuple(k.shape)} and "
                                 f"{tuple(v.shape)}")
    H, D = q.shape[1:]
    K = k.shape[-2]
    _t.check(k.shape[-1] == D, f"k must have q's {D} channels, got {k.shape[-1]}")
    _t.check(8 <= D <= MAX_DIM and D % 8 == 0,
             f"channels must be a multiple of 8 up to {MAX_DIM}, got {D}")
    _t.check(K >= 1 and H >= 1 and H % K == 0,
             f"{H} query heads are not a multiple of {K} key heads")
    return H, K, D


def _options(a, q, scale, cap, slopes):
    D = q.shape[-1]
    a.scale = D ** -0.5 if scale is None else float(scale)
    _t.check(a.scale > 0, f"scale must be positive, got {scale}")
    a.cap = float(cap or 0.0)
    _t.check(a.cap >= 0, f"cap must not be negative, got {cap}")
    if slopes is not None:
        _t.check(isinstance(slopes, Tensor) and slopes.dtype in _t.TYPES
                 and tuple(slopes.shape) == (q.shape[1],) and slopes.device == q.device,
                 f"slopes must be a ({q.shape[1]},) float32 or bfloat16 tensor on {q.device}")
        slopes = slopes.contiguous()
    return slopes


def scene_attention(q: Tensor, k: Tensor, v: Tensor, *, scene_starts: Optional[Tensor] = None,
                    key_starts: Optional[Tensor] = None, longest: Optional[int] = None,
                    causal: bool = False, prefix: Optional[Tensor] = None,
                    scale: Optional[float] = None, cap: float = 0.0,
                    positions: Optional[Tensor] = None, key_positions: Optional[Tensor] = None,
                    slopes: Optional[Tensor] = None, keep: Optional[Tensor] = None) -> Tensor:
    """Attention inside the scenes of a packed batch, differentiable in q, k, v and slopes.

    Args:
        q: (T, H, D); k, v: (N, K, D), H a multiple of K, D a multiple of 8 up to 128.
        scene_starts: (scenes + 1,) int32 first token of each scene; None: one scene.
        key_starts: the same for the keys, where they are not the queries' tokens.
        longest: rows of the longest scene, queries or keys, if known: scenes of one length
            then take fewer workgroups.  It changes no value, but how the slopes' gradient is
            grouped in binary64.
        causal: a token sees the keys up to its own place; where a scene has more keys
            than queries, its queries are the last ones.
        prefix: (scenes,) int32, with causal: leading keys that all tokens of a scene see.
        scale: of the products, 1 / sqrt(D) if None.
        cap: caps the scaled products by cap tanh(. / cap); 0: no cap.
        positions, key_positions: (T, 3), (N, 3) float32 centres, e.g. pos3d or
            pos3d_radii[:, :3]; key_positions default to positions.
        slopes: (H,) float32 or bfloat16: the bias -slopes[h] |p_i - p_j|.
        keep: (N,) int32, bool or uint8: keys with 0 are masked out; num_tiles_hit of the
            projection leaves out culled Gaussians.
    Returns:
        (T, H, D), contiguous.
    """
    if scale != 0 and _native.plain(q, k, v, *_t.present(
            scene_starts, key_starts, prefix, positions, key_positions, slopes, keep)):
        out = _native.scene_attention(q, k, v, scene_starts, key_starts, int(longest or 0),
                                      bool(causal), prefix, float(scale or 0.0), float(cap or 0.0),
                                      positions, key_positions, slopes, keep)
        if out:
            return out[0]
    _t.fixed(positions, "positions", "")
    _t.fixed(key_positions, "key_positions", "")
    return _SceneAttention.apply(q, k, v, slopes, scene_starts, key_starts, prefix, positions,
                                 key_positions, keep, int(longest or 0), bool(causal), scale, cap)


def _point(a, q, k, v, slopes):
    a.q, a.q_row, a.q_head = q.data_ptr(), q.stride(0), q.stride(1)
    a.k, a.k_row, a.k_head = k.data_ptr(), k.stride(-3), k.stride(-2)
    a.v, a.v_row, a.v_head = v.data_ptr(), v.stride(-3), v.stride(-2)
    if slopes is not None:
        a.slopes, a.slopes_dtype = slopes.data_ptr(), _t.TYPES[slopes.dtype]


def _point_packed(a, q, k, v, slopes, q_starts, k_starts, prefix, q_positions, k_positions, keep):
    _point(a, q, k, v, slopes)
    a.q_starts, a.k_starts, a.prefix = _t.ptr(q_starts), _t.ptr(k_starts), _t.ptr(prefix)
    if slopes is not None:
        a.q_positions, a.q_pos_row = q_positions.data_ptr(), q_positions.stride(0)
        a.k_positions, a.k_pos_row = k_positions.data_ptr(), k_positions.stride(0)
    if keep is not None:
        a.keep, a.keep_bytes = keep.data_ptr(), keep.element_size()


def _forward(a, q, k, v, slopes, held, low, lse):
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _point_packed(a, q, k, v, slopes, *held)
    with torch.cuda.device(q.device):
        _t.call("attention_fwd", ctypes.byref(a), out.data_ptr(), _t.ptr(low), _t.ptr(lse),
                _t.stream(q.device))
    return out


def _checked(q, k, v, slopes, scene_starts, key_starts, prefix, positions, key_positions, keep,
             longest, causal, scale, cap):
    """The call's arguments as the kernels take them."""
    H, K, D = _heads(q, k, v, 3)
    dev, T, N = q.device, q.shape[0], k.shape[0]
    _t.check(T <= _t.MAX_TOKENS and N <= _t.MAX_TOKENS, "too many tokens")
    qs, scenes = _t.starts(scene_starts, "scene_starts", dev)
    if key_starts is None:
        _t.check(scenes == 1 or N == T, f"{N} keys for {T} queries need key_starts")
        ks = qs
    else:
        ks, n = _t.starts(key_starts, "key_starts", dev)
        _t.check(n == scenes, f"key_starts hold {n} scenes, scene_starts {scenes}")
    a = _lib.Attention(dtype=_t.TYPES[q.dtype], q_tokens=T, k_tokens=N, heads=H, kv_heads=K, dim=D,
                       scenes=scenes, causal=causal, longest_q=longest, longest_k=longest)
    slopes = _options(a, q, scale, cap, slopes)
    held = [qs, ks, None, None, None, None]
    if prefix is not None:
        _t.check(causal, "prefix needs causal=True")
        held[2] = _t.int32s(prefix, "prefix", scenes, dev)
    if slopes is not None:
        _t.check(positions is not None, "slopes need positions")
        held[3] = _t.positions(positions, "positions", (T, 3), dev)
        if key_positions is None:
            _t.check(N == T, f"{N} keys for {T} queries need key_positions")
            held[4] = held[3]
        else:
            held[4] = _t.positions(key_positions, "key_positions", (N, 3), dev)
    else:
        _t.check(positions is None and key_positions is None, "positions need slopes")
    if keep is not None:
        held[5] = _t.mask(keep, "keep", (N,), dev)
    return a, _t.rows16(q), _t.rows16(k), _t.rows16(v), slopes, held


class _SceneAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, scene_starts, key_starts, prefix, positions, key_positions,
                keep, longest, causal, scale, cap):
        a, q, k, v, slopes, held = _checked(q, k, v, slopes, scene_starts, key_starts, prefix, positions,
                                            key_positions, keep, longest, causal, scale, cap)
        if not any(ctx.needs_input_grad[:4]):
            return _forward(a, q, k, v, slopes, held, None, None)
        lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device)
        # what rounding took from the output: the backward needs it whole
        low = torch.empty(q.shape, dtype=q.dtype, device=q.device) if q.dtype == torch.bfloat16 else None
        out = _forward(a, q, k, v, slopes, held, low, lse)
        ctx.args = a
        ctx.save_for_backward(q, k, v, slopes, out, low, lse, *held)
        return out

    @staticmethod
    @_t.once
    def backward(ctx, dout):
        q, k, v, slopes, out, low, lse, *held = ctx.saved_tensors
        a, dev = ctx.args, q.device
        _point_packed(a, q, k, v, slopes, *held)  # saved-tensor hooks may have moved them
        dout = _t.rows16(dout)
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
        ds = None if slopes is None else torch.empty_like(slopes)
        with torch.cuda.device(dev):
            n = _t.workspace_bytes("attention_bwd_workspace_bytes", a)
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
            _t.call("attention_bwd", ctypes.byref(a), out.data_ptr(), _t.ptr(low),
                    lse.data_ptr(), dout.data_ptr(), dout.stride(0), dout.stride(1), dq.data_ptr(), dk.data_ptr(),
                    dv.data_ptr(), _t.ptr(ds), ws.data_ptr(), n, _t.stream(dev))
        return (dq, dk, dv, ds) + (None,) * 10


def cached_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, lengths: Tensor, *,
                     scale: Optional[float] = None, cap: float = 0.0,
                     positions: Optional[Tensor] = None, key_positions: Optional[Tensor] = None,
                     slopes: Optional[Tensor] = None, keep: Optional[Tensor] = None) -> Tensor:
    """Attention of one new token a scene over its cache; no gradients.

    Args:
        q: (S, H, D); k_cache, v_cache: (S, capacity, K, D), as in `scene_attention`.
        lengths: (S,) int32 live rows of each cache; rows past them are not read.  They
            stay on the device: a captured step may advance them itself.
        positions: (S, 3) float32 of the new tokens; key_positions: (S, capacity, 3).
        keep: (S, capacity) int32, bool or uint8.
        scale, cap, slopes: as in `scene_attention`.
    Returns:
        (S, H, D).
    """
    if scale != 0 and _native.plain(q, k_cache, v_cache, lengths, *_t.present(
            positions, key_positions, slopes, keep)):
        out = _native.cached_attention(q, k_cache, v_cache, lengths, float(scale or 0.0),
                                       float(cap or 0.0), positions, key_positions, slopes, keep)
        if out:
            return out[0]
    for t, what, why in ((q, "q", "s"), (k_cache, "k_cache", "s"), (v_cache, "v_cache", "s"),
                         (positions, "positions", ""), (key_positions, "key_positions", ""),
                         (slopes, "slopes", "")):
        _t.fixed(t, what, why)
    return _CachedAttention.apply(q, k_cache, v_cache, lengths, slopes, positions, key_positions, keep,
                                  scale, cap)


class _CachedAttention(Function):
    @staticmethod
    def forward(ctx, q, k_cache, v_cache, lengths, slopes, positions, key_positions, keep, scale, cap):
        H, K, D = _heads(q, k_cache, v_cache, 4)
        dev, S, N = q.device, q.shape[0], k_cache.shape[1]
        _t.check(k_cache.shape[0] == S, f"k_cache holds {k_cache.shape[0]} scenes, q {S}")
        _t.check(N <= _t.MAX_TOKENS, "too many tokens")
        lengths = _t.int32s(lengths, "lengths", S, dev)
        a = _lib.Attention(dtype=_t.TYPES[q.dtype], q_tokens=S, k_tokens=N, heads=H, kv_heads=K, dim=D,
                           scenes=S)
        slopes = _options(a, q, scale, cap, slopes)
        kp_scene = keep_scene = 0
        if slopes is not None:
            _t.check(positions is not None and key_positions is not None,
                     "slopes need positions and key_positions")
            positions = _t.positions(positions, "positions", (S, 3), dev)
            key_positions = _t.positions(key_positions, "key_positions", (S, N, 3), dev)
            a.q_positions, a.q_pos_row = positions.data_ptr(), positions.stride(0)
            a.k_positions, a.k_pos_row = key_positions.data_ptr(), key_positions.stride(1)
            kp_scene = key_positions.stride(0)
        else:
            _t.check(positions is None and key_positions is None, "positions need slopes")
        if keep is not None:
            keep = _t.mask(keep, "keep", (S, N), dev)
            a.keep, a.keep_bytes, keep_scene = keep.data_ptr(), keep.element_size(), keep.stride(0)
        q, k_cache, v_cache = _t.rows16(q), _t.rows16(k_cache), _t.rows16(v_cache)
        _point(a, q, k_cache, v_cache, slopes)
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        with torch.cuda.device(dev):
            n = _t.workspace_bytes("attention_cached_workspace_bytes", a)
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
            _t.call("attention_cached", ctypes.byref(a), lengths.data_ptr(), k_cache.stride(0),
                    v_cache.stride(0), kp_scene, keep_scene, out.data_ptr(), ws.data_ptr(), n,
                    _t.stream(dev))
        return out

    @staticmethod
    def backward(ctx, dout):
        raise RuntimeError("gs_voxelizer: cached_attention has no gradients")
