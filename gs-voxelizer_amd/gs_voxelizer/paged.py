"""A cache of keys and values in pages, for models that generate tokens of many scenes.

The pools ``k_pages`` and ``v_pages`` (pages, rows, K, D) hold the pages of all scenes; row j of
scene s is row ``j % rows`` of page ``page_table[s, j // rows]``.  A scene so takes the memory of the
rows it has, and grows by a page at a time, wherever one is free.  An entry that names no page
(below 0, or ``pages`` and more) has no rows: they are neither written nor seen.  `append_tokens` writes
new tokens' keys and values, turned by their positions on the way, and `paged_attention` is
`attention.cached_attention` over such a cache.

float32 and bfloat16, no gradients.  Lengths and the table stay on the device, no call reads them on the
host and all calls can be captured in a graph, whose replays then go by what they hold.
"""
import ctypes
from typing import Optional

import torch
from torch import Tensor
from torch.autograd import Function

from . import _lib, _native, _tokens as _t
from .attention import MAX_DIM, _options

PAGE_UNIT = 16  # a page holds a multiple of so many rows


def _pool(t, what, like):
    """A pool, as it is: it is written in place or too large to copy."""
    _t.activations(t, what, 4, like=like)
    P, R, K, D = t.shape
    _t.check(P >= 1 and R >= 1 and R % PAGE_UNIT == 0,
             f"{what} must have pages of a multiple of {PAGE_UNIT} rows, got shape {tuple(t.shape)}")
    _t.check(P < 2**31 and R <= _t.MAX_TOKENS, f"{what} has too many pages or rows")
    _t.check(8 <= D <= MAX_DIM and D % 8 == 0,
             f"channels must be a multiple of 8 up to {MAX_DIM}, got {D}")
    size = t.element_size()
    strides = [s * size if n > 1 else 0 for s, n in zip(t.stride(), t.shape)]
    _t.check(t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % 16 == 0 for s in strides[:-1])
             and strides[1] <= _t.MAX_ROW_BYTES,
             f"{what} must have contiguous channels and rows that start 16-byte aligned, at most 16 MB apart")
    return t


def _is_apart(t, *more):
    """Whether no two elements lie in one place, of a tensor or (more: distance, count) of copies of it."""
    reach = 0
    for stride, n in sorted([(s, n) for s, n in zip(t.stride(), t.shape) if n > 1] + list(more)):
        if stride <= reach:
            return False
        reach += stride * (n - 1)
    return True


def _apart(t, what):
    """Refuses a tensor with several elements in one place, which a kernel would write at once."""
    _t.check(_is_apart(t), f"{what} must not have several elements in one place")


def _share(a, b):
    """Whether two pools of one shape share an element: neither one behind the other nor halves of one pool."""
    a, b = sorted((a, b), key=Tensor.data_ptr)
    by, size = b.data_ptr() - a.data_ptr(), a.element_size()
    if b.data_ptr() >= _span(a)[1]:
        return False
    return a.stride() != b.stride() or by % size != 0 or not _is_apart(a, (by // size, 2))


def _span(t):
    """The memory from a tensor's first element to its last one, in bytes."""
    first = t.data_ptr()
    return first, first + t.element_size() * (1 + sum(s * (n - 1) for s, n in zip(t.stride(), t.shape)))


def _unwritten(t, what, pages, name):
    """Refuses tokens that lie in a pool's memory, where they may change before they are read."""
    if t is not None and pages is not None and t.numel():
        (a, a_end), (b, b_end) = _span(t), _span(pages)
        _t.check(a_end <= b or b_end <= a, f"{what} must not lie in {name}")


def _pages(k_pages, v_pages, page_table, position_pages, keep_pages, like):
    """(the C structure, what it points to): pools, table and what lies beside the keys."""
    _pool(k_pages, "k_pages", like)
    _pool(v_pages, "v_pages", like)
    _t.check(k_pages.shape == v_pages.shape, f"k_pages and v_pages must have one shape, got "
                                             f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    P, R = k_pages.shape[:2]
    dev = like.device
    _t.check(isinstance(page_table, Tensor) and page_table.dtype == torch.int32 and page_table.dim() == 2,
             "page_table must be a 2-D int32 tensor")
    _t.check(page_table.device == dev, f"page_table must be on {dev}, got {page_table.device}")
    _t.check(page_table.shape[1] * R <= _t.MAX_TOKENS, "page_table has room for too many rows")
    table = page_table if page_table.stride(1) == 1 or page_table.shape[1] < 2 else page_table.contiguous()
    p = _lib.Pages(k=k_pages.data_ptr(), v=v_pages.data_ptr(), table=_t.ptr(table), table_row=table.stride(0),
                   pages=P, page_rows=R, table_pages=table.shape[1])
    p.k_page, p.k_row, p.k_head = k_pages.stride()[:3]
    p.v_page, p.v_row, p.v_head = v_pages.stride()[:3]
    if position_pages is not None:
        _t.positions(position_pages, "position_pages", (P, R, 3), dev)
        _t.check(position_pages.stride(-1) == 1, "position_pages must have x, y and z together")
        p.positions, p.pos_page, p.pos_row = (position_pages.data_ptr(), *position_pages.stride()[:2])
    if keep_pages is not None:
        _t.mask(keep_pages, "keep_pages", (P, R), dev)
        _t.check(keep_pages.stride(-1) == 1, "keep_pages must have a page's values together")
        p.keep, p.keep_page, p.keep_bytes = keep_pages.data_ptr(), keep_pages.stride(0), keep_pages.element_size()
    return p, table


def append_tokens(k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, lengths: Tensor, *,
                  q: Optional[Tensor] = None, scene_starts: Optional[Tensor] = None,
                  positions: Optional[Tensor] = None, frequencies: Optional[Tensor] = None,
                  interleaved: bool = False, position_pages: Optional[Tensor] = None,
                  keep: Optional[Tensor] = None, keep_pages: Optional[Tensor] = None) -> Optional[Tensor]:
    """Write new tokens' keys and values to their rows of a cache in pages.

    Of scene s's n new tokens, the i-th becomes row ``lengths[s] - n + i``: lengths count the new
    tokens in, as `paged_attention` then takes them.  A token whose row is below 0 (a scene of
    length 0 that a fixed batch carries along), past the table or in no page is not written; all other rows
    stay as they are.  Two tokens must not have one row (pages that scenes share are only read): what it
    then holds is not said.  As everywhere the last scene ends with the tokens: those that only fill a batch are
    one more scene, of length 0.

    Args:
        k, v: (T, K, D) new tokens, D a multiple of 8 up to 128 (views into one projection's output are taken
            as they are).  No input may lie in the pools' memory.
        k_pages, v_pages: (pages, rows, K, D), rows a multiple of 16, written in place; they may be
            halves of one pool, pool[:, 0] and pool[:, 1].
        page_table: (S, most) int32.
        lengths: (S,) int32 rows of each scene with the new ones.
        q: (T, H, D) queries, turned alike and returned.
        scene_starts: (S + 1,) int32 first token of each scene; None: one token a scene, T = S.
        positions: (T, A) float32; frequencies: (A, P) float32, as `rotary.rotate_qk` takes them.  Without
            frequencies k is written as it is (turned already, or not at all).
        interleaved: pair p is channels (2p, 2p + 1) instead of (p, P + p).
        position_pages: (pages, rows, 3) float32: positions (T, 3) are written there.
        keep, keep_pages: (T,) and (pages, rows), int32, bool or uint8: keep != 0 is written there as 0 or 1,
            e.g. num_tiles_hit of the projection.
    Returns:
        the turned q, contiguous, or None.
    """
    if _native.plain(k, v, k_pages, v_pages, page_table, lengths, *_t.present(
            q, scene_starts, positions, frequencies, position_pages, keep, keep_pages)):
        out = _native.append_tokens(k, v, k_pages, v_pages, page_table, lengths, q, scene_starts, positions,
                                    frequencies, bool(interleaved), position_pages, keep, keep_pages)
        if out:
            return out[0]
    _t.eager("append_tokens")
    for t, what, why in ((k, "k", "s"), (v, "v", "s"), (q, "q", "s"), (k_pages, "k_pages", "s"),
                         (v_pages, "v_pages", "s"), (positions, "positions", ""), (frequencies, "frequencies", ""),
                         (position_pages, "position_pages", "")):
        _t.fixed(t, what, why)
    _t.activations(k, "k", 3)
    _t.activations(v, "v", 3, like=k)
    _t.check(k.shape == v.shape, f"k and v must have one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    T, K, D = k.shape
    dev = k.device
    _t.check(K >= 1, "k must have a head")
    _t.check(T <= _t.MAX_TOKENS, "too many tokens")
    p, table = _pages(k_pages, v_pages, page_table, position_pages, keep_pages, k)
    _t.check(k_pages.shape[2:] == k.shape[1:],
             f"k_pages must have k's {K} heads of {D} channels, got {tuple(k_pages.shape[2:])}")
    for t, what in ((k_pages, "k_pages"), (v_pages, "v_pages"), (position_pages, "position_pages"),
                    (keep_pages, "keep_pages")):
        if t is not None:
            _apart(t, what)
    _t.check(not _share(k_pages, v_pages), "k_pages and v_pages must not share memory")
    S = table.shape[0]
    lengths = _t.int32s(lengths, "lengths", S, dev)
    if scene_starts is None:
        _t.check(S == T, f"{T} tokens for {S} scenes need scene_starts")
    else:
        _t.check(S >= 1, "page_table must have a scene")
        scene_starts = _t.int32s(scene_starts, "scene_starts", S + 1, dev)
    a = _lib.Rotary(dtype=_t.TYPES[k.dtype], tokens=T, kv_heads=K, dim=D, interleaved=bool(interleaved))
    if positions is None:
        _t.check(frequencies is None and position_pages is None, "frequencies and position_pages need positions")
    else:
        _t.check(frequencies is not None or position_pages is not None,
                 "positions need frequencies or position_pages")
        _t.check(isinstance(positions, Tensor) and positions.dtype == torch.float32 and positions.dim() == 2,
                 "positions must be a 2-D float32 tensor")
        _t.check(positions.device == dev, f"positions must be on {dev}, got {positions.device}")
        A = positions.shape[1]
        _t.check(positions.shape[0] == T, f"positions must have {T} rows, got {positions.shape[0]}")
        _t.check(position_pages is None or A == 3, f"position_pages need positions of 3 axes, got {A}")
        a.positions, a.axes = positions.data_ptr(), A
        a.pos_row, a.pos_axis = positions.stride()
    if frequencies is not None:
        _t.check(isinstance(frequencies, Tensor) and frequencies.dtype == torch.float32 and frequencies.dim() == 2,
                 "frequencies must be a 2-D float32 tensor")
        _t.check(frequencies.device == dev, f"frequencies must be on {dev}, got {frequencies.device}")
        _t.check(frequencies.shape[0] == A and 1 <= A <= 8,
                 f"frequencies must have positions' {A} axes, 1 to 8, got {frequencies.shape[0]}")
        P = frequencies.shape[1]
        _t.check(P >= 1 and 2 * P <= D, f"{P} channel pairs do not fit {D} channels")
        frequencies = frequencies.contiguous()
        a.frequencies, a.pairs = frequencies.data_ptr(), P
    out, given_q = None, q
    if q is not None:
        _t.check(frequencies is not None, "q needs frequencies")
        _t.activations(q, "q", 3, like=k)
        _t.check(q.shape[0] == T and q.shape[2] == D and q.shape[1] >= 1,
                 f"q must have k's tokens and channels, got {tuple(q.shape)} for {tuple(k.shape)}")
        q = _t.rows16(q)
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        a.q, a.q_row, a.q_head, a.heads = q.data_ptr(), q.stride(0), q.stride(1), q.shape[1]
    _t.check(K + (0 if q is None else q.shape[1]) <= 4096, "at most 4096 heads")
    _t.check((keep is None) == (keep_pages is None), "keep and keep_pages need each other")
    for pages, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        for t, what in ((k, "k"), (v, "v"), (given_q, "q")):
            _unwritten(t, what, pages, name)
    _unwritten(positions, "positions", position_pages, "position_pages")
    _unwritten(keep, "keep", keep_pages, "keep_pages")
    if keep is not None:
        keep = _t.mask(keep, "keep", (T,), dev)
    k, v = _t.rows16(k), _t.rows16(v)
    a.k, a.k_row, a.k_head = k.data_ptr(), k.stride(0), k.stride(1)
    if T:
        with torch.cuda.device(dev):
            _t.call("paged_append", ctypes.byref(a), v.data_ptr(), v.stride(0), v.stride(1), ctypes.byref(p),
                    lengths.data_ptr(), _t.ptr(scene_starts), S, _t.ptr(keep),
                    0 if keep is None else keep.element_size(), _t.ptr(out), _t.stream(dev))
        _t.written(k_pages, v_pages, position_pages, keep_pages)
    return out


def paged_attention(q: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, lengths: Tensor, *,
                    scale: Optional[float] = None, cap: float = 0.0, positions: Optional[Tensor] = None,
                    position_pages: Optional[Tensor] = None, slopes: Optional[Tensor] = None,
                    keep_pages: Optional[Tensor] = None) -> Tensor:
    """Attention of one new token a scene over its pages; no gradients.

    Args:
        q: (S, H, D); k_pages, v_pages: (pages, rows, K, D), H a multiple of K, D a multiple of 8 up to
            128, rows a multiple of 16.
        page_table: (S, most) int32; entries past a scene's last row are not read.  Scenes may share pages.
        lengths: (S,) int32 live rows of each scene, at most ``most * rows`` (more are left out); rows past them
            are not read, and a scene without any gives 0.
        positions: (S, 3) float32 of the new tokens; position_pages: (pages, rows, 3).
        keep_pages: (pages, rows) int32, bool or uint8: keys with 0 are masked out.
        scale, cap, slopes: as in `attention.scene_attention`.
    Returns:
        (S, H, D).
    """
    if scale != 0 and _native.plain(q, k_pages, v_pages, page_table, lengths, *_t.present(
            positions, position_pages, slopes, keep_pages)):
        out = _native.paged_attention(q, k_pages, v_pages, page_table, lengths, float(scale or 0.0),
                                      float(cap or 0.0), positions, position_pages, slopes, keep_pages)
        if out:
            return out[0]
    for t, what, why in ((q, "q", "s"), (k_pages, "k_pages", "s"), (v_pages, "v_pages", "s"),
                         (positions, "positions", ""), (position_pages, "position_pages", ""),
                         (slopes, "slopes", "")):
        _t.fixed(t, what, why)
    return _PagedAttention.apply(q, k_pages, v_pages, page_table, lengths, slopes, positions, position_pages,
                                 keep_pages, scale, cap)


class _PagedAttention(Function):
    @staticmethod
    def forward(ctx, q, k_pages, v_pages, page_table, lengths, slopes, positions, position_pages, keep_pages, scale,
                cap):
        _t.activations(q, "q", 3)
        dev, (S, H, D) = q.device, q.shape
        p, table = _pages(k_pages, v_pages, page_table, position_pages, keep_pages, q)
        K = k_pages.shape[2]
        _t.check(k_pages.shape[3] == D, f"k_pages must have q's {D} channels, got {k_pages.shape[3]}")
        _t.check(K >= 1 and H >= 1 and H % K == 0, f"{H} query heads are not a multiple of {K} key heads")
        _t.check(table.shape[0] == S, f"page_table holds {table.shape[0]} scenes, q {S}")
        lengths = _t.int32s(lengths, "lengths", S, dev)
        q = _t.rows16(q)
        a = _lib.Attention(dtype=_t.TYPES[q.dtype], q_tokens=S, heads=H, kv_heads=K, dim=D, scenes=S,
                           q=q.data_ptr(), q_row=q.stride(0), q_head=q.stride(1))
        slopes = _options(a, q, scale, cap, slopes)
        if slopes is not None:
            _t.check(positions is not None and position_pages is not None,
                     "slopes need positions and position_pages")
            positions = _t.positions(positions, "positions", (S, 3), dev)
            a.slopes, a.slopes_dtype = slopes.data_ptr(), _t.TYPES[slopes.dtype]
            a.q_positions, a.q_pos_row = positions.data_ptr(), positions.stride(0)
        else:
            _t.check(positions is None and position_pages is None, "positions need slopes")
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        with torch.cuda.device(dev):
            n = ctypes.c_size_t(0)
            _t.call("attention_paged_workspace_bytes", ctypes.byref(a), ctypes.byref(p), ctypes.byref(n))
            ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
            _t.call("attention_paged", ctypes.byref(a), ctypes.byref(p), lengths.data_ptr(), out.data_ptr(),
                    ws.data_ptr(), n.value, _t.stream(dev))
        return out

    @staticmethod
    def backward(ctx, dout):
        raise RuntimeError("gs_voxelizer: paged_attention has no gradients")
