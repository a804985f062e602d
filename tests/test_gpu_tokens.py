"""The operators on packed tokens: views, batches and routes that the operators' own files leave out."""
import pytest
import torch

import token_reference as R
from gs_voxelizer import _native, attention, gated_norm, rotary

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])


@pytest.fixture(params=["native", "python"])
def route(request, monkeypatch):
    """Through the native autograd nodes where they take the call, and through the Python classes."""
    if request.param == "python":
        monkeypatch.setattr(_native, "available", False)
    else:
        assert _native.available
    return request.param


def _gen(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


@TYPES
def test_one_token_out_of_a_long_array(device, route, dtype):
    """q, k, v and the gradient of a scene's one token, sliced out of arrays of 20,000: the strides of
    their one row, 20 MB and more, mean nothing."""
    g, H, D = _gen(device, 0), 8, 64
    long = torch.zeros(4, 1, 20_000, H, D, dtype=dtype, device=device)
    long[:, :, 7] = torch.randn(4, 1, H, D, generator=g, device=device).to(dtype)
    q, k, v, dout = (t[:, 7].requires_grad_() for t in long)
    assert q.stride(0) * q.element_size() > 1 << 24
    out = attention.scene_attention(q, k, v)
    got = torch.autograd.grad(out, (q, k, v), dout)
    assert torch.equal(out, v) and torch.equal(got[2], dout)
    assert not got[0].any() and not got[1].any()
    with torch.no_grad():
        n = torch.tensor([1], dtype=torch.int32, device=device)
        cache = v.detach()[:, None].expand(1, 1, H, D)
        assert torch.equal(attention.cached_attention(q, cache, cache, n), v)
        pos, f = torch.rand(1, 3, device=device), rotary.axis_frequencies((11, 11, 10), device=device)
        a, b = rotary.rotate_qk(q, k, pos, f), rotary.rotate_qk(q.clone(), k.clone(), pos, f)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        w = torch.ones(D, device=device)
        a = gated_norm.gated_residual_norm(q[:, 0], k[:, 0], w)
        b = gated_norm.gated_residual_norm(q[:, 0].clone(), k[:, 0].clone(), w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@TYPES
def test_one_head_of_an_odd_width(device, route, dtype):
    """A head axis of one entry may have any stride."""
    g = _gen(device, 1)
    wide = torch.randn(3, 30, 1, 72, generator=g, device=device).to(dtype)
    q, k, v = (t.as_strided((30, 1, 64), (72, 5, 1)) for t in wide)
    got = attention.scene_attention(q, k, v)
    assert torch.equal(got, attention.scene_attention(q.clone(), k.clone(), v.clone()))
