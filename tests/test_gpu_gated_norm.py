"""gated_residual_norm against its definition in binary64; gradients from torch's
differentiation of that definition.  Bounds: binary32 sums of C terms are off by at most
C 2^-24 of their terms' sizes, so a row's values and gradients by (2 C + 64) 2^-24 of the sizes
that they are made of, and sums over rows by as much again for each row; then one rounding
to the tensor's type."""
import pytest
import torch

import token_reference as R
from gs_voxelizer import _native, gated_norm

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(autouse=True, params=["native", "python"])
def route(request, monkeypatch):
    """Through the native autograd nodes where they take the call, and through the Python classes."""
    if request.param == "python":
        monkeypatch.setattr(_native, "available", False)
    else:
        assert _native.available
LEAVES = ("x", "branch", "weight", "branch_weight", "scale", "gate")


def _case(device, T, C, lengths=None, types=(F32, F32), gate="scene", gate_type=None, norm=True,
          scale=True, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape, s=1.0, mean=0.0, t=F32):
        return (torch.randn(shape, generator=g, device=device) * s + mean).to(t)

    c = dict(x=normal(T, C, t=types[0]), branch=normal(T, C, s=3.0, t=types[1]),
             weight=normal(C, s=0.2, mean=1.0), branch_weight=normal(C, s=0.2, mean=1.0) if norm else None,
             scale=normal(C, s=0.1, mean=0.5) if scale else None, gate=None, starts=None,
             dy=normal(T, C, t=types[0]), dh=normal(T, C, t=types[1]))
    if lengths:
        c["starts"] = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)],
                                   dtype=torch.int32, device=device)
    if gate:
        rows = {"scene": len(lengths) if lengths else 1, "token": T, "one": 1}[gate]
        c["gate"] = normal(rows, C, s=0.5, mean=1.0, t=gate_type or types[1])
    return c


def _run(c, train=True, **more):
    v = {n: None if c[n] is None else c[n].detach().clone().requires_grad_(train) for n in LEAVES}
    y, h = gated_norm.gated_residual_norm(
        v["x"], v["branch"], v["weight"], branch_weight=v["branch_weight"], scale=v["scale"],
        gate=v["gate"], scene_starts=c["starts"], eps=1e-5, **more)
    got = {"y": y.detach(), "h": h.detach()}
    if train:
        names = [n for n in LEAVES if v[n] is not None]
        got.update(zip(names, torch.autograd.grad((y, h), [v[n] for n in names], (c["dy"], c["dh"]))))
    return got


def _reference(c):
    T, C = c["x"].shape
    v = {n: None if c[n] is None else c[n].detach().double().requires_grad_() for n in LEAVES}
    dev = c["x"].device
    if v["gate"] is None:
        gate = torch.ones(T, C, dtype=torch.float64, device=dev)
        scene = torch.zeros(T, dtype=torch.int64, device=dev)
    elif c["starts"] is not None:
        scene = torch.searchsorted(c["starts"][1:-1].contiguous(),
                                   torch.arange(T, device=dev, dtype=torch.int32), right=True)
        gate = v["gate"][scene]
    else:
        scene = (torch.arange(T, device=dev) if c["gate"].shape[0] == T
                 else torch.zeros(T, dtype=torch.int64, device=dev))
        gate = v["gate"][scene]

    def rstd(t):
        return (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt()

    rb = rstd(v["branch"]) if v["branch_weight"] is not None else None
    n = v["branch"] if rb is None else v["branch"] * rb * v["branch_weight"]
    by = gate if v["scale"] is None else gate * v["scale"]
    y = v["x"] + by * n
    ry = rstd(y)
    h = y * ry * v["weight"]
    names = [n_ for n_ in LEAVES if v[n_] is not None]
    grads = dict(zip(names, torch.autograd.grad((y, h), [v[n_] for n_ in names],
                                                (c["dy"].double(), c["dh"].double()))))
    with torch.no_grad():
        e = 2.0 ** -24 * (2 * C + 64)
        u = {n_: R.ROUND[c[n_].dtype] for n_ in names}
        size_y = v["x"].abs() + (by * n).abs()
        w, bw = v["weight"].abs(), 1.0 if rb is None else v["branch_weight"].abs()
        tol = {"y": u["x"] * y.abs() + e * size_y,
               "h": u["branch"] * h.abs() + e * (size_y * ry * w + 2 * h.abs() + (
                   (size_y * y.abs()).mean(-1, keepdim=True) * ry ** 2 * h.abs()))}
        # what y_hat and dy' may be off by, in units of e
        yh = (y * ry).abs()
        o_yh = size_y * ry + 2 * yh + (size_y * y.abs()).mean(-1, keepdim=True) * ry ** 2 * yh
        t = c["dh"].double().abs() * w
        dy1 = grads["x"]
        o_dy = c["dy"].double().abs() + 2 * ry * (
            t + yh * (t * yh).mean(-1, keepdim=True) * 3 + o_yh * (t * yh).mean(-1, keepdim=True)
            + yh * (t * o_yh).mean(-1, keepdim=True)) + (
            ry * (t + yh * (t * yh).mean(-1, keepdim=True)) * (size_y * y.abs()).mean(-1, keepdim=True) * ry ** 2)
        tol["x"] = u["x"] * dy1.abs() + e * o_dy
        fh = (v["branch"] if rb is None else v["branch"] * rb).abs()
        g_dn = by.abs() * bw
        o_u = (o_dy + 4 * dy1.abs()) * g_dn
        if rb is None:
            o_b = o_u
        else:
            uu = dy1.abs() * g_dn
            o_b = rb * (o_u + 4 * uu + fh * ((o_u + 6 * uu) * fh).mean(-1, keepdim=True))
        tol["branch"] = u["branch"] * grads["branch"].abs() + e * o_b
        rows = 2.0 ** -24 * (T + 64)
        dh = c["dh"].double().abs()
        o_a = (e * (o_dy + 4 * dy1.abs()) + rows * dy1.abs()) * fh
        tol["weight"] = u["weight"] * grads["weight"].abs() + ((e * o_yh + rows * yh) * dh).sum(0)
        if v["scale"] is not None:
            tol["scale"] = u["scale"] * grads["scale"].abs() + (o_a * gate.abs() * bw).sum(0)
        if rb is not None:
            tol["branch_weight"] = u["branch_weight"] * grads["branch_weight"].abs() + (
                o_a * by.abs()).sum(0)
        if v["gate"] is not None:
            s = 1.0 if v["scale"] is None else v["scale"].abs()
            tol["gate"] = (u["gate"] * grads["gate"].abs()
                           + torch.zeros_like(v["gate"]).index_add_(0, scene, o_a * s * bw))
    return {"y": y.detach(), "h": h.detach(), **grads}, tol


def _check(c, **more):
    val, tol = _reference(c)
    got = _run(c, **more)
    assert set(got) == set(val)
    for n in got:
        like = {"y": "x", "h": "branch"}.get(n, n)
        assert got[n].dtype == c[like].dtype and got[n].is_contiguous(), n
        R.assert_within(got[n], val[n], tol[n], n)
    return got


TYPES = [(F32, F32), (F32, BF16), (BF16, BF16)]


@pytest.mark.parametrize("types", TYPES, ids=["f32", "mixed", "bf16"])
@pytest.mark.parametrize("channels", [1, 3, 64, 250, 333, 500, 512, 513, 1024, 1100, 2048, 2500, 8192])
def test_channels(device, types, channels):
    _check(_case(device, 37, channels, [20, 0, 1, 16], types))


@pytest.mark.parametrize("types", TYPES, ids=["f32", "mixed", "bf16"])
@pytest.mark.parametrize("lengths", [[1], [0, 0, 2], [1000], [1, 700, 0, 33, 66], [5] * 130], ids=str)
def test_scenes(device, types, lengths):
    _check(_case(device, sum(lengths), 96, lengths, types))


@pytest.mark.parametrize("types", TYPES, ids=["f32", "mixed", "bf16"])
@pytest.mark.parametrize("gate", [None, "one", "token", "scene"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("scale", [False, True])
def test_options(device, types, gate, norm, scale):
    _check(_case(device, 300, 128, [130, 170] if gate == "scene" else None, types, gate=gate, norm=norm,
                 scale=scale))
    if gate and types[1] == BF16:
        _check(_case(device, 40, 128, [13, 27] if gate == "scene" else None, types, gate=gate,
                     gate_type=F32, norm=norm, scale=scale))


def test_many_rows(device):
    _check(_case(device, 30_001, 250, [29_000, 1_001], (F32, BF16)))


def test_hints_views_and_repeats(device):
    """Any `longest`, rows of a wider buffer, rows off alignment, another stream: the same bits for
    row results; sums over rows are split by `longest` and agree within their bound."""
    c = _case(device, 403, 256, [100, 3, 300], (F32, BF16))
    want = _check(c)
    for longest in (None, 1, 300, 10**6):
        got = _check(c, longest=longest)
        for n in ("y", "h", "x", "branch"):
            assert torch.equal(got[n], want[n]), (longest, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(c)
    torch.cuda.current_stream().wait_stream(side)
    for n in got:
        assert torch.equal(got[n], want[n]), n
    for pad in (8, 1):
        d = dict(c)
        for n in ("x", "branch", "gate", "dy", "dh"):
            wide = torch.zeros(c[n].shape[0], 256 + pad + 3 * (pad == 8), dtype=c[n].dtype, device=device)
            d[n] = wide[:, pad:pad + 256].copy_(c[n])
        v = {n: d[n].detach().requires_grad_() for n in ("x", "branch", "gate")}
        y, h = gated_norm.gated_residual_norm(v["x"], v["branch"], c["weight"],
                                              branch_weight=c["branch_weight"], scale=c["scale"],
                                              gate=v["gate"], scene_starts=c["starts"], eps=1e-5)
        got = torch.autograd.grad((y, h), list(v.values()), (d["dy"], d["dh"]))
        val, tol = _reference(c)
        for n, t in zip(("y", "h", "x", "branch", "gate"), (y, h) + got):
            R.assert_within(t.detach(), val[n], tol[n], n)


def test_one_output_used(device):
    """Only h, or only y, takes part in the loss."""
    c = _case(device, 90, 64, [50, 40])
    for keep in ("dy", "dh"):
        d = dict(c)
        other = "dh" if keep == "dy" else "dy"
        d[other] = torch.zeros_like(c[other])
        val, tol = _reference(d)
        v = {n: c[n].detach().clone().requires_grad_() for n in LEAVES}
        y, h = gated_norm.gated_residual_norm(v["x"], v["branch"], v["weight"],
                                              branch_weight=v["branch_weight"], scale=v["scale"],
                                              gate=v["gate"], scene_starts=c["starts"], eps=1e-5)
        (y if keep == "dy" else h).backward(c[keep])
        for n in LEAVES:
            R.assert_within(v[n].grad, val[n], tol[n], n)


def test_gradients_against_differences(device):
    c = _case(device, 40, 48, [25, 15])
    got = _run(c)
    g, step = torch.Generator(device=device).manual_seed(7), 2.0 ** -6
    for n in LEAVES:
        way = torch.randn(c[n].shape, generator=g, device=device)
        ends = []
        for sign in (1, -1):
            r = _run(dict(c, **{n: c[n] + sign * step * way}), train=False)
            ends.append((r["y"].double() * c["dy"].double()).sum()
                        + (r["h"].double() * c["dh"].double()).sum())
        slope = float(ends[0] - ends[1]) / (2 * step)
        parts = got[n].double() * way.double()
        # float32 results near 1 over the step, and third derivatives of some units times its square
        assert abs(slope - float(parts.sum())) <= 0.02 * float(parts.square().sum().sqrt()) + 0.02, n


def test_zero_rows_and_empty_batch(device):
    c = _case(device, 12, 64, [12])
    c["x"][:6] = 0
    c["branch"][:6] = 0
    got = _check(c)
    assert not got["h"][:6].any()
    c = _case(device, 0, 64, [0, 0])
    got = _run(c)
    for n in ("weight", "branch_weight", "scale", "gate"):
        assert got[n].shape == c[n].shape and not got[n].any()


def test_refusals(device):
    x = torch.zeros(6, 32, device=device)
    w = torch.ones(32, device=device)
    starts = torch.tensor([0, 2, 6], dtype=torch.int32, device=device)

    def refused(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            gated_norm.gated_residual_norm(*args, **kw)

    refused("CUDA", x.cpu(), x, w)
    refused("float32 or bfloat16", x.half(), x, w)
    refused("bfloat16 where x is", x.bfloat16(), x, w)
    refused("x's shape", x, x[:5], w)
    refused("weight must be", x, x, w[:31])
    refused("weight must be", x, x, w.bfloat16())
    refused("scale must be", x, x, w, scale=w.double())
    refused("branch_weight must be", x, x, w, branch_weight=w[None])
    refused("gate must have a row", x, x, w, gate=x[:3], scene_starts=starts)
    refused("gate must have a row", x, x, w, gate=x[:4])
    refused("gate must be", x, x, w, gate=x.bfloat16())
    refused("int32", x, x, w, scene_starts=starts.long())
    refused("eps", x, x, w, eps=-1.0)
    big = torch.zeros(1, 8193, device=device)
    refused("channels", big, big, big[0])


def test_gradients_are_not_differentiated_again(device):
    x = torch.ones(5, 32, device=device, requires_grad=True)
    y, h = gated_norm.gated_residual_norm(x, torch.ones_like(x), torch.ones(32, device=device))
    g, = torch.autograd.grad((y + h).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate"):
        g.sum().backward()


def test_saved_tensor_hooks_may_move_what_is_saved(device):
    """Saved tensors kept in host memory between the passes: the same gradients."""
    c = _case(device, 300, 128, [130, 170], (F32, BF16))
    want = _run(c)
    with torch.autograd.graph.save_on_cpu():
        got = _run(c)
    for n in got:
        assert torch.equal(got[n], want[n]), n
