"""The cache in pages and the optimiser's step without a GPU: what their C entries accept and refuse."""
import ctypes

import pytest

from gs_voxelizer import _lib, _tokens

OK, INVALID, WORKSPACE, SIZE_OVERFLOW = 0, 1, 3, 4
MAX = _tokens.MAX_TOKENS


def _pages(**more):
    a = dict(k=1024, v=2048, k_page=16 * 128, k_row=128, k_head=64, v_page=16 * 128, v_row=128, v_head=64,
             table=4096, table_row=8, pages=9, page_rows=16, table_pages=8)
    return _lib.Pages(**dict(a, **more))


def _query(**more):
    a = dict(dtype=1, q_tokens=4, heads=4, kv_heads=2, dim=64, scenes=4, scale=0.125, q=1024, q_row=256, q_head=64)
    return _lib.Attention(**dict(a, **more))


def _plan(a, p):
    n = ctypes.c_size_t(0)
    return _lib.load().gsv_attention_paged_workspace_bytes(ctypes.byref(a), ctypes.byref(p), ctypes.byref(n)), n.value


@pytest.mark.parametrize("more", [
    dict(page_rows=0), dict(page_rows=8), dict(page_rows=24), dict(page_rows=-16), dict(pages=0), dict(pages=-1),
    dict(table_pages=-1), dict(table_row=-1), dict(k=1032), dict(v=2056), dict(k=None), dict(k_row=129),
    dict(v_head=65), dict(k_row=-128), dict(v_row=1 << 24), dict(keep=4096, keep_bytes=2)])
def test_pages_that_are_refused(more):
    assert _plan(_query(), _pages())[0] == OK
    assert _plan(_query(), _pages(**more))[0] == INVALID


@pytest.mark.parametrize("more", [
    dict(dim=4), dict(dim=136), dict(dim=20), dict(heads=3), dict(kv_heads=0), dict(dtype=2), dict(scale=0.0),
    dict(cap=-1.0), dict(causal=1), dict(q_tokens=5), dict(scenes=-1, q_tokens=-1), dict(slopes=1024),
    dict(slopes=1024, slopes_dtype=1, q_positions=1024)])
def test_queries_that_are_refused(more):
    assert _plan(_query(**more), _pages())[0] == INVALID


def test_rows_and_scenes_that_are_too_many():
    assert _plan(_query(), _pages(table_pages=MAX // 16))[0] == OK
    assert _plan(_query(), _pages(table_pages=MAX // 16 + 1))[0] == SIZE_OVERFLOW
    assert _plan(_query(), _pages(table_pages=2**31 - 1, page_rows=2**31 - 16))[0] == SIZE_OVERFLOW
    assert _plan(_query(scenes=1 << 21, q_tokens=1 << 21), _pages())[0] == OK
    assert _plan(_query(scenes=(1 << 21) + 1, q_tokens=(1 << 21) + 1), _pages())[0] == SIZE_OVERFLOW
    assert _plan(_query(scenes=1 << 20, q_tokens=1 << 20, heads=16), _pages())[0] == SIZE_OVERFLOW


@pytest.mark.parametrize("scenes", [1, 2, 16, 65, 300, 5000])
@pytest.mark.parametrize("table_pages", [0, 1, 8, 9, 200, 20_000])
@pytest.mark.parametrize("dtype,dim", [(0, 32), (0, 128), (1, 40), (1, 64), (1, 128)])
def test_the_workspace_holds_a_row_for_each_part(scenes, table_pages, dtype, dim):
    """Parts are one for each scene and at most a round of workgroups more; none where a scene is a step or two."""
    st, n = _plan(_query(scenes=scenes, q_tokens=scenes, dtype=dtype, dim=dim), _pages(table_pages=table_pages))
    assert st == OK
    if table_pages * 16 <= 64:
        assert n == 0
    elif n:
        rows, rest = divmod(n - 8 * scenes, 4 * dim + 8)
        assert rest == 0 and rows % 4 == 0
        assert scenes < rows // 4 <= scenes + 1024


def test_a_workspace_that_is_too_small_is_refused():
    a, p = _query(), _pages(table_pages=1000)
    st, n = _plan(a, p)
    assert st == OK and n > 0
    assert _lib.load().gsv_attention_paged(ctypes.byref(a), ctypes.byref(p), 1024, 1024, 1024, n - 1, None) == WORKSPACE
    assert _lib.load().gsv_attention_paged(ctypes.byref(a), ctypes.byref(p), None, 1024, 1024, n, None) == INVALID
    assert _lib.load().gsv_attention_paged(ctypes.byref(a), ctypes.byref(p), 1024, 1032, 1024, n, None) == INVALID
    assert _lib.load().gsv_attention_paged(ctypes.byref(a), ctypes.byref(p), 1024, 1024, 1032, n, None) == INVALID
    assert _lib.load().gsv_attention_paged(ctypes.byref(a), ctypes.byref(_pages(table_pages=1000, table=None)), 1024,
                                           1024, 1024, n, None) == INVALID


def _append(p=None, v=1024, v_row=128, v_head=64, lengths=1024, starts=None, scenes=4, keep=None, keep_bytes=0,
            q_out=1024, **more):
    r = dict(dtype=1, tokens=4, heads=4, kv_heads=2, dim=64, pairs=32, axes=3, q=1024, k=1024, q_row=256, q_head=64,
             k_row=128, k_head=64, positions=1024, frequencies=1024, pos_row=3, pos_axis=1)
    r = _lib.Rotary(**dict(r, **more))
    return _lib.load().gsv_paged_append(ctypes.byref(r), v, v_row, v_head, ctypes.byref(p or _pages()), lengths,
                                        starts, scenes, keep, keep_bytes, q_out, None)


@pytest.mark.parametrize("more", [
    dict(dtype=2), dict(tokens=-1), dict(tokens=5), dict(scenes=5), dict(heads=-1), dict(kv_heads=0), dict(dim=4),
    dict(dim=60), dict(dim=136), dict(pairs=33), dict(pairs=-1), dict(pairs=0), dict(axes=0), dict(axes=9),
    dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(lengths=None), dict(positions=None),
    dict(frequencies=None), dict(k=1032), dict(v=1032), dict(q_out=1032), dict(v_row=129), dict(v_head=65),
    dict(k_row=129), dict(q_head=65), dict(keep=1024, keep_bytes=1), dict(heads=4095),
    dict(p=_pages(keep=1024, keep_bytes=1)), dict(p=_pages(keep=1024, keep_bytes=1), keep=1024, keep_bytes=3),
    dict(p=_pages(keep=1024, keep_bytes=2), keep=1024, keep_bytes=1), dict(p=_pages(positions=1024), axes=2),
    dict(p=_pages(positions=1024), heads=0, pairs=0, positions=None), dict(p=_pages(page_rows=20)),
    dict(p=_pages(pages=0)), dict(p=_pages(k=1032)), dict(p=_pages(v_page=2049)), dict(p=_pages(k_row=129)),
    dict(p=_pages(table=None)), dict(p=_pages(v=None)), dict(starts=1024, scenes=0)])
def test_tokens_that_are_refused(more):
    assert _append(**more) == INVALID


def test_more_tokens_than_are_taken():
    assert _append(tokens=MAX + 1, scenes=MAX + 1) == SIZE_OVERFLOW
    assert _append(p=_pages(table_pages=MAX // 16 + 1)) == SIZE_OVERFLOW
    assert _append(tokens=0, scenes=0) == OK  # nothing to do: nothing is launched


def _adamw(tensors, **more):
    all = (_lib.AdamwTensor * max(len(tensors), 1))(*tensors)
    a = _lib.Adamw(tensors=ctypes.addressof(all), count=len(tensors),
                   **dict(dict(beta1=0.9, beta2=0.999, eps=1e-8), **more))
    n = ctypes.c_size_t(0)
    st = _lib.load().gsv_adamw_workspace_bytes(ctypes.byref(a), ctypes.byref(n))
    return a, all, st, n.value


def _tensor(at=0, n=100, **more):
    t = dict(param=1 << 20, grad=2 << 20, exp_avg=3 << 20, exp_avg_sq=4 << 20, numel=n, step=1, lr=1e-3)
    t = {k: x + at if x >= 1 << 20 else x for k, x in t.items()}
    return _lib.AdamwTensor(**dict(t, **more))


@pytest.mark.parametrize("more", [
    dict(numel=-1), dict(step=0), dict(dtype=2), dict(grad_dtype=2), dict(master=5 << 20), dict(param=None),
    dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(param=(1 << 20) + 2), dict(exp_avg=(1 << 20) + 1),
    dict(dtype=1, param=(1 << 20) + 1), dict(dtype=1, master=(1 << 20) + 2), dict(lr_device=(1 << 20) + 2)])
def test_tensors_of_a_step_that_are_refused(more):
    assert _adamw([_tensor()])[2] == OK
    assert _adamw([_tensor(), _tensor(1 << 12, **more)])[2] == INVALID


@pytest.mark.parametrize("more", [dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0), dict(eps=-1.0),
                                  dict(eps=float("nan")), dict(max_norm=-1.0), dict(beta2=float("nan")), dict(count=-1)])
def test_steps_that_are_refused(more):
    assert _adamw([_tensor()], **{k: v for k, v in more.items() if k != "count"})[2] == (
        INVALID if "count" not in more else OK)
    a, _, _, _ = _adamw([_tensor()])
    a.count = more.get("count", 1)
    n = ctypes.c_size_t(0)
    assert _lib.load().gsv_adamw_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == (
        INVALID if "count" in more else OK)


def test_a_step_of_too_many_elements_is_refused():
    assert _adamw([_tensor(n=(1 << 34) + 1)])[2] == SIZE_OVERFLOW
    assert _adamw([_tensor(n=1 << 34), _tensor(n=1)])[2] == SIZE_OVERFLOW


def test_a_step_s_workspace():
    assert _adamw([_tensor()])[3] == 0
    assert _adamw([_tensor()], counter=1024)[3] == 16
    a, _, _, n = _adamw([_tensor(n=10_000), _tensor(1 << 16, n=1)], max_norm=1.0)
    assert n == 16 + 8 * (2 + 1)  # a sum for each 8,192 elements of a tensor
    assert _lib.load().gsv_adamw(ctypes.byref(a), 1024, n - 1, None) == WORKSPACE
    assert _lib.load().gsv_adamw(ctypes.byref(a), None, n, None) == INVALID


@pytest.mark.parametrize("second", [
    dict(param=(1 << 20) + 396), dict(exp_avg=3 << 20), dict(exp_avg_sq=(4 << 20) - 396), dict(exp_avg=(1 << 20) + 4),
    dict(param=(6 << 20), exp_avg=6 << 20), dict(dtype=1, master=(4 << 20) + 396), dict(grad=(1 << 20) + 396),
    dict(grad=(4 << 20) - 396), dict(grad_dtype=1, grad=(3 << 20) - 198)])
def test_tensors_that_share_memory_are_refused(second):
    """(Before anything is launched: these addresses are nobody's.)"""
    a, _all, st, _ = _adamw([_tensor(), _tensor(1 << 16, **second)])
    assert st == OK
    assert _adamw([_tensor(), _tensor(1 << 16)])[2] == OK
    assert _lib.load().gsv_adamw(ctypes.byref(a), None, 0, None) == INVALID
