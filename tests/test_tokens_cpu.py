"""The operators on packed tokens without a GPU: what their host side accepts, copies and refuses."""
import ctypes

import pytest
import torch

import token_rounding as T
from gs_voxelizer import _lib, _tokens

OK, SIZE_OVERFLOW = 0, 4
F32, BF16 = torch.float32, torch.bfloat16


def _attention(**more):
    a = dict(dtype=1, q_tokens=64, k_tokens=64, heads=4, kv_heads=4, dim=64, scenes=1, scale=0.125,
             q=1024, k=1024, v=1024)
    for n in "qkv":
        a[n + "_row"], a[n + "_head"] = 256, 64
    return _lib.Attention(**dict(a, **more))


def _plan(name, a):
    """The status of a call's host side: a workspace's size needs no device."""
    return getattr(_lib.load(), f"gsv_attention_{name}_workspace_bytes")(
        ctypes.byref(a), ctypes.byref(ctypes.c_size_t(0)))


def _one_token(dtype=BF16):
    """A scene's token sliced out of an array of 20,000: (1, H, D), its rows 40 MB apart."""
    return torch.zeros(1, 20_000, 16, 64, dtype=dtype)[:, 7]


def test_strides_of_one_entry_mean_nothing():
    assert _plan("bwd", _attention()) == OK
    for n in "qkv":
        assert _plan("bwd", _attention(q_tokens=1, k_tokens=1, **{n + "_row": 20_480_000})) == OK
        assert _plan("bwd", _attention(q_tokens=1, k_tokens=1, **{n + "_row": 7})) == OK
        assert _plan("bwd", _attention(heads=1, kv_heads=1, **{n + "_head": 7})) == OK
        assert _plan("bwd", _attention(**{n + "_row": 20_480_000})) != OK
        assert _plan("bwd", _attention(**{n + "_row": 257})) != OK
        assert _plan("bwd", _attention(**{n + "_head": 65})) != OK
    assert _plan("cached", _attention(q_tokens=1, scenes=1, q_row=20_480_000)) == OK


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_views_are_taken_as_they_are_or_copied(dtype):
    one = _one_token(dtype)
    assert _tokens.rows16(one) is one
    head = torch.zeros(5, 1, 67, dtype=dtype)[..., :64]
    odd = head.as_strided((1, 1, 64), (7, 3, 1))
    assert _tokens.rows16(odd) is odd
    # rows off alignment, far rows, a strided last axis, a start off alignment: canonical copies
    far = torch.zeros(2, 1 << 24, dtype=dtype)[:, :256].unflatten(1, (4, 64))
    for t in (head, far, torch.zeros(5, 64, 4, dtype=dtype).transpose(1, 2),
              torch.zeros(65, dtype=dtype)[1:].view(1, 1, 64)):
        c = _tokens.rows16(t)
        assert c is not t and c.is_contiguous() and c.stride() == (t.shape[1] * 64, 64, 1)
        assert c.data_ptr() % 16 == 0 and torch.equal(c, t)


@pytest.mark.parametrize("tokens", [2**31 - 2**16 + 1, 2**31 - 64, 2**31 - 1])
def test_counts_that_would_pass_int32_are_refused(tokens):
    """Kernels step past the last row by up to 2^15 rows: counts nearer to 2^31 would wrap there, and a
    loop over keys would not end.  (No pointers: nothing could be launched.)"""
    L = _lib.load()
    assert _plan("bwd", _attention(q_tokens=tokens)) == SIZE_OVERFLOW
    assert _plan("bwd", _attention(k_tokens=tokens)) == SIZE_OVERFLOW
    assert _plan("cached", _attention(k_tokens=tokens, scenes=64)) == SIZE_OVERFLOW
    n = _lib.Norm(dtype=0, branch_dtype=0, tokens=tokens, channels=1, scenes=1, eps=1e-6)
    assert L.gsv_gated_norm_fwd(ctypes.byref(n), None, None, None) == SIZE_OVERFLOW
    n.tokens, n.scenes = 5, tokens
    assert L.gsv_gated_norm_fwd(ctypes.byref(n), None, None, None) == SIZE_OVERFLOW
    r = _lib.Rotary(dtype=0, tokens=tokens, heads=1, kv_heads=0, dim=2, pairs=1, axes=1)
    assert L.gsv_rotary(ctypes.byref(r), None, None, 0, None) == SIZE_OVERFLOW
    # the most that is taken
    assert _plan("bwd", _attention(k_tokens=_tokens.MAX_TOKENS)) == OK
    assert _plan("cached", _attention(k_tokens=_tokens.MAX_TOKENS, scenes=64)) == OK
    r.tokens = _tokens.MAX_TOKENS
    assert L.gsv_rotary(ctypes.byref(r), None, None, 0, None) == 1  # its pointers are missing


def _bwd_bytes(**more):
    n = ctypes.c_size_t(0)
    a = _attention(**more)
    assert _lib.load().gsv_attention_bwd_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == OK
    return n.value


@pytest.mark.parametrize("longest", [0, 1, 128, 16_000, 64_000, -5])
def test_launches_go_by_the_rows_and_scenes_there_are(longest):
    """The workspace holds a binary64 sum for each workgroup of the rows' kernel: their number is at most
    a tile for each 128 rows and one for each scene, whatever is known of the longest scene."""
    more = dict(q_tokens=64_000, k_tokens=64_000, heads=8, kv_heads=8, scenes=500, longest_q=longest,
                longest_k=longest, q_starts=1024, k_starts=1024)
    plain = _bwd_bytes(**more)
    n = (_bwd_bytes(**more, slopes=1024, q_positions=1024, k_positions=1024) - plain) / (8 * 8)
    assert 0 < n <= 64_000 // 128 + 500


def test_more_scenes_than_a_launch_holds_are_refused():
    more = dict(heads=64, kv_heads=64, q_starts=1024, k_starts=1024)
    assert _plan("bwd", _attention(scenes=1 << 29, **more)) == OK
    assert _plan("bwd", _attention(scenes=(1 << 29) + 1, **more)) == SIZE_OVERFLOW
    more["heads"] = more["kv_heads"] = 1 << 14
    assert _plan("bwd", _attention(scenes=1 << 29, **more)) == SIZE_OVERFLOW


@pytest.mark.parametrize("longest", [0, 1, 2_900, 20_000])
def test_the_norm_s_partial_sums_go_by_the_rows_and_scenes_there_are(longest):
    n = ctypes.c_size_t(0)
    a = _lib.Norm(dtype=0, branch_dtype=0, tokens=20_000, channels=1024, scenes=7, longest=longest, eps=1e-6,
                  starts=1024, x=1024, branch=1024, weight=1024, x_row=1024, branch_row=1024)
    assert _lib.load().gsv_gated_norm_bwd_workspace_bytes(ctypes.byref(a), ctypes.byref(n)) == OK
    assert n.value <= 2 * 4 * 1024 * (1024 + 7)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_the_bounds_tell_a_lost_part_of_out_and_the_rows_rests(dim, causal):
    """The bounds of the GPU tests, on the oracle with the kernels' roundings: they hold, and fail where D
    comes from the rounded output alone, or the rows' rests stay in the slopes' gradient."""
    found = 0
    for seed in range(4):
        args, want = T.clear_winners(450, dim, seed, causal)
        right = T.rounded_head(*args)
        for n in ("out", "dq", "dk", "dv"):
            T.assert_rounded_twice(right[n], want[n], n)
        assert T.off(right["dslopes"], want["dslopes"]) <= T.SLOPES
        wrong = T.rounded_head(*args, whole_out=False)
        for n in ("dq", "dk"):
            assert T.off(wrong[n], want[n]) > T.rounded_twice(want[n])
        wrong = T.rounded_head(*args, rests=False)
        found += T.off(wrong["dslopes"], want["dslopes"]) > T.SLOPES
    assert found >= 3
