"""rotate_qk against its definition in binary64, elementwise: an angle formed in binary64, its
sine and cosine off by at most 2^-22 (the reduced angle's rounding, 2^-24 pi, and the
functions'), and one rounding to the tensor's type."""
import pytest
import torch

import token_reference as R
from gs_voxelizer import _native, rotary

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(autouse=True, params=["native", "python"])
def route(request, monkeypatch):
    """Through the native autograd nodes where they take the call, and through the Python classes."""
    if request.param == "python":
        monkeypatch.setattr(_native, "available", False)
    else:
        assert _native.available


def _gen(device, seed=0):
    return torch.Generator(device=device).manual_seed(seed)


def _turned(x, positions, frequencies, interleaved, sign=1):
    P = frequencies.shape[1]
    theta = (positions.double()[:, :, None] * frequencies.double()).sum(1)[:, None] * sign
    x = x.double()
    a, b = ((x[..., 0:2 * P:2], x[..., 1:2 * P:2]) if interleaved
            else (x[..., :P], x[..., P:2 * P]))
    both = a * theta.cos() - b * theta.sin(), a * theta.sin() + b * theta.cos()
    size = a.abs() + b.abs()
    if interleaved:
        head, size = torch.stack(both, -1).flatten(-2), size.repeat_interleave(2, -1)
    else:
        head, size = torch.cat(both, -1), torch.cat((size, size), -1)
    rest = x[..., 2 * P:]
    return torch.cat((head, rest), -1), torch.cat((size, torch.zeros_like(rest)), -1)


def _check(got, x, positions, frequencies, interleaved, sign=1):
    val, size = _turned(x, positions, frequencies, interleaved, sign)
    assert got.dtype == x.dtype and got.is_contiguous()
    R.assert_within(got, val, R.ROUND[x.dtype] * val.abs() + 2.0 ** -22 * size + 1e-30, "rotary")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,dim,pairs", [
    (1, 1, 1, 2, 1), (1, 8, 2, 64, 32), (3, 3, 1, 16, 5), (130, 12, 4, 40, 18), (1000, 2, 2, 128, 64),
    (77, 5, 5, 41, 20), (5000, 4, 1, 32, 12), (64, 1, 1, 1024, 512), (10, 300, 1, 6, 3)])
def test_forward_and_backward(device, dtype, interleaved, tokens, heads, kv, dim, pairs):
    g = _gen(device)
    q, k, dq, dk = (torch.randn(tokens, n, dim, generator=g, device=device).to(dtype)
                    for n in (heads, kv, heads, kv))
    pos = 256 * torch.rand(tokens, 4, generator=g, device=device)[:, :3] - 20
    f = rotary.axis_frequencies([pairs // 3 + (a < pairs % 3) for a in range(3)], device=device)
    q.requires_grad_(), k.requires_grad_()
    a, b = rotary.rotate_qk(q, k, pos, f, interleaved=interleaved)
    _check(a.detach(), q.detach(), pos, f, interleaved)
    _check(b.detach(), k.detach(), pos, f, interleaved)
    ga, gb = torch.autograd.grad((a, b), (q, k), (dq, dk))
    _check(ga, dq, pos, f, interleaved, -1)
    _check(gb, dk, pos, f, interleaved, -1)


@pytest.mark.parametrize("axes", [1, 2, 4, 8])
def test_axes_and_slanted_frequencies(device, axes):
    """Any number of axes; pairs that turn with several of them."""
    g = _gen(device, 1)
    q = torch.randn(33, 2, 32, generator=g, device=device)
    pos = 100 * torch.randn(33, axes, generator=g, device=device)
    f = torch.randn(axes, 16, generator=g, device=device)
    a, none = rotary.rotate_qk(q, None, pos, f)
    assert none is None
    _check(a, q, pos, f, False)


def test_large_angles(device):
    """A million radians: the angle is still formed exactly enough."""
    g = _gen(device, 2)
    q = torch.randn(50, 2, 8, generator=g, device=device)
    pos = 1e6 * torch.rand(50, 1, generator=g, device=device)
    f = torch.ones(1, 4, device=device)
    # 2^-52 of the angle in turns, over 2^-22: nothing
    _check(rotary.rotate_qk(q, None, pos, f)[0], q, pos, f, False)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_views(device, dtype, interleaved):
    """Views into a projection, rows off alignment by an element, strided last axis, an expanded
    gradient: the bits of contiguous tensors."""
    g = _gen(device, 3)
    qkv = torch.randn(99, 8, 48, generator=g, device=device).to(dtype)
    pos = 50 * torch.rand(99, 3, generator=g, device=device)
    f = rotary.axis_frequencies((8, 8, 8), device=device)
    q, k = qkv[:, :4], qkv[:, 4:6]
    want = rotary.rotate_qk(q.contiguous(), k.contiguous(), pos, f, interleaved)
    for a, b in (((q, k)), (torch.cat((q[:, :, :1], q), 2)[..., 1:], torch.cat((k[..., :3], k), 2)[..., 3:]),
                 (q.transpose(1, 2).contiguous().transpose(1, 2), k)):
        got = rotary.rotate_qk(a, b, pos, f, interleaved)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    wide = torch.zeros(99, 7, device=device)
    wide[:, ::3] = pos
    got = rotary.rotate_qk(q, k, wide[:, ::3], f, interleaved)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x = q.detach().clone().requires_grad_()
    a, b = rotary.rotate_qk(x, k, pos, f, interleaved)
    one, = torch.autograd.grad(a, x, torch.ones((), dtype=dtype, device=device).expand(a.shape),
                               retain_graph=True)
    two, = torch.autograd.grad(a, x, torch.ones_like(a))
    assert torch.equal(one, two)


def test_scores_depend_on_relative_positions(device):
    """q.k after the turn is the same when all positions move together (float32: angles to 300,
    64 products of size 1, each off by 2^-21)."""
    g = _gen(device, 4)
    q, k = (torch.randn(40, 1, 64, generator=g, device=device) for _ in "qk")
    pos = 100 * torch.rand(40, 3, generator=g, device=device)
    f = rotary.axis_frequencies((11, 11, 10), device=device)

    def scores(p):
        a, b = rotary.rotate_qk(q, k, p, f)
        return a[:, 0].double() @ b[:, 0].double().T

    # positions move by whole numbers, exactly: 2^-17 is their spacing at 100
    pos = (pos * 2 ** 16).round() / 2 ** 16
    assert float((scores(pos) - scores(pos + 64)).abs().max()) < 64 * 8 * 2.0 ** -21


def test_empty_and_partial_gradients(device):
    f = rotary.axis_frequencies((2, 1, 1), device=device)
    z = torch.zeros(0, 2, 8, device=device)
    a, b = rotary.rotate_qk(z, z, torch.zeros(0, 3, device=device), f)
    assert a.shape == b.shape == z.shape
    g = _gen(device, 5)
    q, k = (torch.randn(9, 2, 8, generator=g, device=device) for _ in "qk")
    pos = torch.rand(9, 3, generator=g, device=device)
    k.requires_grad_()
    a, b = rotary.rotate_qk(q, k, pos, f)
    (a.sum() + (2 * b).sum()).backward()  # q takes no gradient
    _check(k.grad, torch.full_like(k, 2.0).detach(), pos, f, False, -1)


def test_refusals(device):
    q = torch.zeros(5, 2, 8, device=device)
    pos = torch.zeros(5, 3, device=device)
    f = rotary.axis_frequencies((2, 1, 1), device=device)

    def refused(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            rotary.rotate_qk(*args, **kw)

    refused("CUDA", q.cpu(), q, pos, f)
    refused("float32 or bfloat16", q.half(), None, pos, f)
    refused("must be torch.float32", q, q.bfloat16(), pos, f)
    refused("3 axes", q[0], None, pos, f)
    refused("tokens and channels", q, q[:4], pos, f)
    refused("positions must have shape", q, q, pos[:, :2], f)
    refused("float32", q, q, pos.double(), f)
    refused("float32", q, q, pos, f.double())
    refused("do not fit", q[..., :6], None, pos, f)
    refused("detach", q, q, pos.clone().requires_grad_(), f)
    with pytest.raises(ValueError):
        rotary.axis_frequencies([])


def test_gradients_are_not_differentiated_again(device):
    q = torch.ones(5, 2, 8, device=device, requires_grad=True)
    f = rotary.axis_frequencies((2, 1, 1), device=device)
    a, b = rotary.rotate_qk(q, q, torch.ones(5, 3, device=device), f)
    g, = torch.autograd.grad((a.sum() + b.sum()), q, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate"):
        g.sum().backward()
