"""What the attention operators take as scale and cap, without a GPU."""
import ctypes

import pytest

from gs_voxelizer import _lib

OK, INVALID = 0, 1
INF = float("inf")


@pytest.mark.parametrize("more,status", [
    (dict(cap=0.0), OK), (dict(cap=1e30), OK), (dict(cap=INF), INVALID), (dict(cap=-INF), INVALID), (dict(cap=1e39), INVALID),
    (dict(cap=float("nan")), INVALID), (dict(scale=INF), INVALID), (dict(scale=1e39), INVALID),
    (dict(scale=float("nan")), INVALID)])
def test_scale_and_cap(more, status):
    """Infinities are refused: every score would be NaN."""
    a = dict(dtype=1, q_tokens=4, heads=4, kv_heads=2, dim=64, scenes=4, scale=0.125, q=1024, q_row=256, q_head=64)
    pages = _lib.Pages(k=1024, v=2048, k_page=16 * 128, k_row=128, k_head=64, v_page=16 * 128, v_row=128, v_head=64,
                       table=4096, table_row=8, pages=9, page_rows=16, table_pages=8)
    n = ctypes.c_size_t(0)
    L = _lib.load()
    query = _lib.Attention(**dict(a, **more))
    assert L.gsv_attention_paged_workspace_bytes(ctypes.byref(query), ctypes.byref(pages), ctypes.byref(n)) == status
    cached = _lib.Attention(**dict(a, k=1024, v=2048, k_row=128, k_head=64, v_row=128, v_head=64, k_tokens=100, **more))
    assert L.gsv_attention_cached_workspace_bytes(ctypes.byref(cached), ctypes.byref(n)) == status
