"""scene_attention and cached_attention against their definition in binary64: every element
within a bound made of the roundings that the operators document (token_reference.py)."""
import pytest
import torch

import token_reference as R
from gs_voxelizer import _native, attention

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(autouse=True, params=["native", "python"])
def route(request, monkeypatch):
    """Through the native autograd nodes where they take the call, and through the Python classes."""
    if request.param == "python":
        monkeypatch.setattr(_native, "available", False)
    else:
        assert _native.available
NAMES = ("dq", "dk", "dv", "dslopes")


def _gen(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def _case(device, dtype, lengths, H, K, D, seed=0, key_lengths=None, bias=False, culled=0.0,
          causal=False, prefix=False, cap=0.0, slopes_dtype=None, spread=40.0):
    g = _gen(device, seed)
    T, N = sum(lengths), sum(key_lengths or lengths)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=device).to(dtype)

    def starts(ls):
        return torch.tensor([sum(ls[:i]) for i in range(len(ls) + 1)], dtype=torch.int32,
                            device=device)

    c = dict(q=normal(T, H, D), k=normal(N, K, D), v=normal(N, K, D), dout=normal(T, H, D),
             q_starts=starts(lengths), k_starts=starts(key_lengths) if key_lengths else None,
             causal=causal, cap=cap)
    if prefix:
        c["prefix"] = torch.tensor([n // 3 for n in (key_lengths or lengths)], dtype=torch.int32,
                                   device=device)
    if bias:
        c["q_positions"] = spread * torch.rand(T, 3, generator=g, device=device)
        c["k_positions"] = (spread * torch.rand(N, 3, generator=g, device=device) if key_lengths
                            else c["q_positions"])
        c["slopes"] = torch.tensor([2.0 ** -(h + 1) for h in range(H)], device=device).to(
            slopes_dtype or dtype)
    if culled:
        c["keep"] = (torch.rand(N, generator=g, device=device) >= culled).int() * 3
    return c


def _run(c, train=True, **more):
    leaves = [c[n].detach().clone().requires_grad_(train) for n in ("q", "k", "v")]
    slopes = c.get("slopes")
    if slopes is not None:
        slopes = slopes.detach().clone().requires_grad_(train)
    out = attention.scene_attention(
        *leaves, scene_starts=c["q_starts"], key_starts=c["k_starts"], causal=c["causal"],
        prefix=c.get("prefix"), cap=c["cap"], positions=c.get("q_positions"),
        key_positions=c.get("k_positions"), slopes=slopes, keep=c.get("keep"), **more)
    got = {"out": out.detach()}
    if train:
        out.backward(c["dout"])
        got.update(dq=leaves[0].grad, dk=leaves[1].grad, dv=leaves[2].grad)
        if slopes is not None:
            got["dslopes"] = slopes.grad
    return got


def _check(c, what, **more):
    val, tol = R.attention(**{n: t for n, t in c.items()})
    got = _run(c, **more)
    for n, t in got.items():
        assert t.dtype == (c["slopes"].dtype if n == "dslopes" else c["q"].dtype)
        R.assert_within(t, val[n], tol[n], f"{what} {n}")
    return got


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("lengths", [[1], [2, 1], [31, 0, 33], [64], [65, 127, 1, 0, 128], [129, 300]],
                         ids=str)
@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
def test_lengths(device, dtype, lengths, bias):
    _check(_case(device, dtype, lengths, 2, 1, 64, bias=bias), f"{lengths}")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(1, 1), (3, 3), (6, 2), (8, 1)], ids=str)
@pytest.mark.parametrize("dim", [8, 24, 32, 40, 64, 72, 96, 128])
def test_heads_and_channels(device, dtype, heads, dim):
    _check(_case(device, dtype, [100, 57], *heads, dim, bias=True, causal=True, cap=20.0),
           f"{heads} {dim}")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("causal,prefix", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("culled", [0.0, 0.4])
def test_masks_and_cap(device, dtype, causal, prefix, cap, culled):
    _check(_case(device, dtype, [200, 3, 131], 4, 2, 32, bias=True, causal=causal, prefix=prefix,
                 cap=cap, culled=culled), "masks")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,key_lengths", [([5, 70], [150, 40]), ([0, 9, 1], [4, 0, 300]),
                                                 ([130], [1])], ids=str)
def test_other_keys(device, dtype, causal, lengths, key_lengths):
    """Keys of another count than the queries: rows without keys among them."""
    _check(_case(device, dtype, lengths, 4, 4, 64, key_lengths=key_lengths, bias=True,
                 causal=causal), "other keys")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_rows_without_keys_are_zero(device, dtype):
    c = _case(device, dtype, [40, 90], 2, 2, 32, bias=True)
    c["keep"] = torch.ones(130, dtype=torch.bool, device=device)
    c["keep"][:40] = False
    got = _check(c, "empty")
    assert not got["out"][:40].any() and not got["dq"][:40].any()
    assert not got["dk"][:40].any() and not got["dv"][:40].any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf")])
def test_masked_keys_reach_nothing(device, dtype, junk):
    """Whatever k, v and the positions of culled keys hold, the results are those without it."""
    c = _case(device, dtype, [70, 200], 4, 2, 64, bias=True, culled=0.3, cap=8.0, key_lengths=[90, 171])
    want = _run(c)
    for n in ("k", "v", "k_positions"):
        c[n] = c[n].clone()
        c[n][c["keep"] == 0] = junk
    got = _run(c)
    for n in got:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_large_scores(device, dtype):
    """Scores of some thousands: the softmax is a maximum, nothing overflows."""
    c = _case(device, dtype, [150], 2, 2, 64)
    c["q"], c["k"] = c["q"] * 30, c["k"] * 30
    val, _ = R.attention(**c)
    got = _run(c)
    for n in got:
        assert torch.isfinite(got[n]).all(), n
    # rows whose best key leads by 30: every other weight is below e^-30 (a score is off by
    # 2^-24 times its 64 products, below 0.1), so the row is that key's value, with the weight,
    # its product, the sum's reciprocal and the result each rounded once
    t = torch.einsum("qhd,khd->hqk", c["q"].double().cpu(), c["k"].double().cpu()) / 8
    best = t.topk(2, dim=-1)
    clear = (best.values[..., 0] - best.values[..., 1] > 30).T.to(device)
    assert int(clear.sum()) > 100
    pick = torch.stack([c["v"][best.indices[h, :, 0].to(device), h] for h in range(2)], 1)
    off = (got["out"].double() - pick.double()).abs()[clear]
    assert bool((off <= 4 * R.ROUND[dtype] * pick.double().abs()[clear] + 1e-9).all())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_long_scene(device, dtype):
    _check(_case(device, dtype, [2500], 2, 1, 64, bias=True, causal=True, prefix=True), "long")


def test_slopes_keep_their_type(device):
    _check(_case(device, BF16, [90, 33], 3, 1, 64, bias=True, slopes_dtype=F32), "f32 slopes")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_strided_views_and_hints(device, dtype):
    """Views into one projection's output, (N, 4) position rows, any `longest`, an expanded
    gradient: the same bits as contiguous tensors."""
    c = _case(device, dtype, [140, 61], 4, 2, 32, bias=True, causal=True, prefix=True)
    want = _run(c)
    T = 201
    qkv = torch.cat([c["q"], c["k"], c["v"]], 1).requires_grad_()
    pos = torch.cat([c["q_positions"], torch.zeros(T, 1, device=device)], 1)
    for longest in (None, 1, 64, 140, 5000):
        q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
        out = attention.scene_attention(q, k, v, scene_starts=c["q_starts"], longest=longest,
                                        causal=True, prefix=c["prefix"], positions=pos[:, :3],
                                        slopes=c["slopes"])
        assert torch.equal(out, want["out"])
        g, = torch.autograd.grad(out, qkv, c["dout"])
        for n, part in zip(("dq", "dk", "dv"), (g[:, :4], g[:, 4:6], g[:, 6:])):
            assert torch.equal(part, want[n]), (longest, n)
    # rows that are not 16-byte aligned, heads before tokens, an expanded gradient
    odd = torch.zeros(T, 4, 37, dtype=dtype, device=device)[:, :, 1:33].copy_(c["q"])
    swapped = c["k"].transpose(0, 1).contiguous().transpose(0, 1)
    with torch.no_grad():
        out = attention.scene_attention(odd, swapped, c["v"], scene_starts=c["q_starts"],
                                        causal=True, prefix=c["prefix"],
                                        positions=c["q_positions"], slopes=c["slopes"])
    assert torch.equal(out, want["out"])
    q = c["q"].clone().requires_grad_()
    out = attention.scene_attention(q, c["k"], c["v"])
    a, = torch.autograd.grad(out, q, torch.ones((), dtype=dtype, device=device).expand(out.shape),
                             retain_graph=True)
    b, = torch.autograd.grad(out, q, torch.ones_like(out))
    assert torch.equal(a, b)


def test_repeats_are_bit_equal_and_streams(device):
    c = _case(device, BF16, [500, 20, 333], 8, 2, 64, bias=True, culled=0.1)
    want = _run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(c)
    torch.cuda.current_stream().wait_stream(side)
    for n in got:
        assert torch.equal(got[n], want[n]), n


def test_starts_out_of_range_stay_inside(device):
    """Starts are clamped to the arrays: whatever they hold, every access stays inside."""
    c = _case(device, BF16, [50, 60, 70], 2, 2, 32)
    want = _run(c)
    c["q_starts"][0], c["q_starts"][3] = -7, 1 << 30
    got = _run(c)
    for n in got:
        assert torch.equal(got[n], want[n]), n
    c["q_starts"][1], c["q_starts"][2] = 1 << 30, -5
    for n, t in _run(c).items():
        assert t.shape == want[n].shape


def test_gradients_against_differences(device):
    """The directional derivative of a float32 loss, by central differences."""
    c = _case(device, F32, [60, 45], 4, 2, 32, bias=True, causal=True, prefix=True, cap=6.0, culled=0.1)
    got = _run(c)
    g, step = _gen(device, 9), 2.0 ** -6
    for n in ("q", "k", "v", "slopes"):
        way = torch.randn(c[n].shape, generator=g, device=device)
        ends = []
        for sign in (1, -1):
            d = dict(c)
            d[n] = c[n] + sign * step * way
            ends.append((_run(d, train=False)["out"].double() * c["dout"].double()).sum())
        slope = float(ends[0] - ends[1]) / (2 * step)
        want = float((got["d" + n].double() * way.double()).sum())
        # outputs near 1 with errors of some 2^-22, 13440 of them with random signs, over the
        # step, and the third derivative (some units) times its square
        size = float((got["d" + n].double() * way.double()).square().sum().sqrt())
        assert abs(slope - want) <= 0.02 * size + 0.02, (n, slope, want)


# ---- one token over a cache


def _cache(device, dtype, lengths, capacity, H, K, D, seed=0, bias=True, culled=0.0):
    g = _gen(device, seed)
    S = len(lengths)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=device).to(dtype)

    c = dict(q=normal(S, H, D), k=normal(S, capacity, K, D), v=normal(S, capacity, K, D),
             lengths=torch.tensor(lengths, dtype=torch.int32, device=device), pos=None, kpos=None,
             slopes=None, keep=None)
    if bias:
        c["pos"] = 40 * torch.rand(S, 3, generator=g, device=device)
        c["kpos"] = 40 * torch.rand(S, capacity, 3, generator=g, device=device)
        c["slopes"] = torch.tensor([2.0 ** -(h + 1) for h in range(H)], device=device).to(dtype)
    if culled:
        c["keep"] = torch.rand(S, capacity, generator=g, device=device) >= culled
    return c


def _cached(c, cap):
    return attention.cached_attention(c["q"], c["k"], c["v"], c["lengths"], cap=cap,
                                      positions=c["pos"], key_positions=c["kpos"],
                                      slopes=c["slopes"], keep=c["keep"])


def _cached_reference(c, cap):
    vals, tols = [], []
    for s, n in enumerate(c["lengths"].clamp(0, c["k"].shape[1]).tolist()):
        bias = c["slopes"] is not None
        val, tol = R.attention(
            c["q"][s:s + 1], c["k"][s, :n], c["v"][s, :n], cap=cap, slopes=c["slopes"],
            q_positions=c["pos"][s:s + 1] if bias else None,
            k_positions=c["kpos"][s, :n] if bias else None,
            keep=None if c["keep"] is None else c["keep"][s, :n])
        vals.append(val["out"])
        tols.append(tol["out"])
    return torch.cat(vals), torch.cat(tols)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads", [(1, 1), (8, 2), (12, 4), (40, 1)], ids=str)
@pytest.mark.parametrize("dim", [8, 32, 40, 64, 96, 128])
def test_cached_heads_and_channels(device, dtype, heads, dim):
    c = _cache(device, dtype, [0, 1, 31, 33, 300], 300, *heads, dim)
    R.assert_within(_cached(c, 0.0), *_cached_reference(c, 0.0), f"{heads} {dim}")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("culled", [0.0, 0.5, 1.0])
def test_cached_masks(device, dtype, cap, bias, culled):
    c = _cache(device, dtype, [129, 5000, 64, 4097], 5000, 4, 2, 64, bias=bias, culled=culled)
    got = _cached(c, cap)
    R.assert_within(got, *_cached_reference(c, cap), "masks")
    if culled == 1.0:
        assert not got.any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_cached_rows_past_the_length_are_not_read(device, dtype, junk):
    c = _cache(device, dtype, [0, 7, 130, 700], 1000, 4, 2, 64, culled=0.2)
    want = _cached(c, 6.0)
    dead = torch.arange(1000, device=device)[None] >= c["lengths"][:, None]
    dead |= ~c["keep"]
    for n in ("k", "v", "kpos"):
        c[n][dead] = junk
    assert torch.equal(_cached(c, 6.0), want)
    c["lengths"][3] = 1 << 30  # clamped to the capacity
    c["lengths"][0] = -3
    _cached(c, 6.0)


def test_cached_equals_the_last_row_of_a_scene(device):
    """The two entry points agree: a causal scene's last token, and one query over its keys."""
    c = _case(device, F32, [777], 6, 3, 64, bias=True, causal=True)
    whole = _run(c, train=False)["out"]
    got = attention.cached_attention(
        c["q"][-1:], c["k"][None], c["v"][None], torch.tensor([777], dtype=torch.int32, device=device),
        positions=c["q_positions"][-1:], key_positions=c["k_positions"][None], slopes=c["slopes"])
    val, tol = R.attention(c["q"][-1:], c["k"], c["v"], slopes=c["slopes"],
                           q_positions=c["q_positions"][-1:], k_positions=c["k_positions"])
    R.assert_within(got, val["out"], tol["out"], "cached")
    R.assert_within(whole[-1:], val["out"], tol["out"], "whole")


def test_cached_views_of_a_larger_cache(device):
    """Strided scenes, rows and heads, and a capacity that is a slice of a longer buffer."""
    c = _cache(device, BF16, [100, 37], 256, 4, 2, 64)
    want = _cached(c, 0.0)
    big = torch.full((2, 400, 2, 2, 64), float("nan"), dtype=BF16, device=device)
    big[:, :256, 0], big[:, :256, 1] = c["k"], c["v"]
    d = dict(c, k=big[:, :256, 0], v=big[:, :256, 1])
    assert torch.equal(_cached(d, 0.0), want)


def test_cached_row_offsets_past_32_bits(device):
    """A cache whose last rows lie beyond 2^32 elements: only those rows are live keys."""
    K, D, N = 4, 128, (1 << 32) // 512 + 64
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    k = torch.zeros(1, N, K, D, dtype=BF16, device=device)
    v = torch.zeros(1, N, K, D, dtype=BF16, device=device)
    g = _gen(device, 3)
    k[0, -64:] = torch.randn(64, K, D, generator=g, device=device).to(BF16)
    v[0, -64:] = torch.randn(64, K, D, generator=g, device=device).to(BF16)
    keep = torch.zeros(1, N, dtype=torch.bool, device=device)
    keep[0, -64:] = True
    q = torch.randn(1, 8, D, generator=g, device=device).to(BF16)
    got = attention.cached_attention(q, k, v, torch.tensor([N], dtype=torch.int32, device=device),
                                     keep=keep)
    val, tol = R.attention(q, k[0, -64:], v[0, -64:])
    R.assert_within(got, val["out"], tol["out"], "far rows")


# ---- refusals, before anything is launched


def _refused(match, call, *args, **kw):
    with pytest.raises(ValueError, match=match):
        call(*args, **kw)


def test_refusals(device):
    q = torch.zeros(10, 4, 64, device=device)
    k = torch.zeros(10, 2, 64, device=device)
    f = attention.scene_attention
    pos, slopes = torch.zeros(10, 3, device=device), torch.zeros(4, device=device)
    _refused("CUDA", f, q.cpu(), k, k)
    _refused("float32 or bfloat16", f, q.half(), k.half(), k.half())
    _refused("must be torch.float32", f, q, k.bfloat16(), k)
    _refused("3 axes", f, q[0], k, k)
    _refused("one shape", f, q, k, k[:5])
    _refused("64 channels", f, q, k[..., :32], k[..., :32])
    _refused("multiple of 8", f, q[..., :12], k[..., :12], k[..., :12])
    _refused("multiple of 8", f, *(torch.zeros(4, 1, 136, device=device) for _ in range(3)))
    _refused("not a multiple of", f, q[:, :3], k, k)
    _refused("scale", f, q, k, k, scale=0.0)
    _refused("cap", f, q, k, k, cap=-1.0)
    _refused("need positions", f, q, k, k, slopes=slopes)
    _refused("need slopes", f, q, k, k, positions=pos)
    _refused("positions", f, q, k, k, slopes=slopes, positions=pos[:9])
    _refused("slopes must be", f, q, k, k, slopes=slopes[:3], positions=pos)
    _refused("detach", f, q, k, k, slopes=slopes, positions=pos.clone().requires_grad_())
    _refused("keep", f, q, k, k, keep=torch.ones(10, device=device))
    _refused("keep", f, q, k, k, keep=torch.ones(9, device=device, dtype=torch.bool))
    _refused("causal", f, q, k, k, prefix=torch.zeros(1, dtype=torch.int32, device=device))
    _refused("int32", f, q, k, k, scene_starts=torch.zeros(3, device=device, dtype=torch.int64))
    _refused("scenes", f, q, k, k, scene_starts=torch.zeros(3, device=device, dtype=torch.int32),
             key_starts=torch.zeros(2, device=device, dtype=torch.int32))
    _refused("key_starts", f, q[:5], k, k,
             scene_starts=torch.zeros(3, device=device, dtype=torch.int32))
    _refused("key_positions", f, q[:5], k, k, slopes=slopes, positions=pos[:5])


def test_cached_refusals(device):
    q = torch.zeros(3, 4, 64, device=device)
    k = torch.zeros(3, 20, 2, 64, device=device)
    n = torch.zeros(3, dtype=torch.int32, device=device)
    f = attention.cached_attention
    _refused("4 axes", f, q, k[0], k[0], n)
    _refused("scenes", f, q[:2], k, k, n[:2])
    _refused("lengths", f, q, k, k, n[:2])
    _refused("int32", f, q, k, k, n.long())
    _refused("detach", f, q.requires_grad_(), k, k, n)
    with torch.no_grad():
        assert f(q, k, k, n).shape == q.shape
    _refused("key_positions", f, q.detach(), k, k, n, slopes=torch.zeros(4, device=device),
             positions=torch.zeros(3, 3, device=device))


def test_empty_batches(device):
    z = torch.zeros(0, 2, 32, device=device, requires_grad=True)
    out = attention.scene_attention(z, z, z)
    assert out.shape == z.shape
    out.sum().backward()
    assert z.grad.shape == z.shape
    q = torch.zeros(4, 2, 32, device=device, requires_grad=True)
    out = attention.scene_attention(q, z, z)
    assert not out.any()
    out.sum().backward()
    assert not q.grad.any()
    q = torch.ones(2, 2, 32, device=device)
    cache = torch.zeros(2, 0, 2, 32, device=device)
    assert not attention.cached_attention(q, cache, cache, torch.zeros(2, dtype=torch.int32,
                                                                       device=device)).any()


def test_captured_cached_step(device):
    """A decode step in a HIP graph advances its lengths itself; each replay equals the eager call."""
    c = _cache(device, BF16, [40, 100], 256, 4, 2, 64)
    q = c["q"].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _cached(c, 0.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _cached(c, 0.0)
        c["lengths"].add_(1)
    c["lengths"].copy_(torch.tensor([40, 100], dtype=torch.int32))
    for step in range(4):
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        d = dict(c, lengths=torch.tensor([40 + step, 100 + step], dtype=torch.int32, device=device))
        assert torch.equal(got, _cached(d, 0.0)), step
        c["q"].copy_(q * (step + 2))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [(1, 1), (8, 1)], ids=str)
def test_key_gradients_summed_over_parts(device, dtype, dim, heads):
    """Few key tiles and many rows: several workgroups share a key tile's rows."""
    _check(_case(device, dtype, [40, 1500], *heads, dim, bias=True, causal=True, prefix=True,
                 key_lengths=[60, 900]), "parts")


def test_gradients_are_not_differentiated_again(device):
    c = _case(device, F32, [20], 2, 2, 32)
    q = c["q"].requires_grad_()
    g, = torch.autograd.grad(attention.scene_attention(q, c["k"], c["v"]).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate"):
        g.sum().backward()


def test_saved_tensor_hooks_may_move_what_is_saved(device):
    c = _case(device, BF16, [150, 77], 4, 2, 64, bias=True, causal=True, prefix=True, culled=0.2)
    want = _run(c)
    with torch.autograd.graph.save_on_cpu():
        got = _run(c)
    for n in got:
        assert torch.equal(got[n], want[n]), n


# ---- the kernels of larger calls: those above have few enough rows that the waves of a workgroup
# share them; two hundred scenes of one token more, or long scenes of many heads, are past that


MANY = [1] * 200


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dim", [8, 24, 32, 40, 64, 72, 96, 128])
@pytest.mark.parametrize("heads", [(1, 1), (4, 2)], ids=str)
def test_many_scenes(device, dtype, dim, heads):
    _check(_case(device, dtype, [33, 0, 140, 1] + MANY, *heads, dim, bias=True, causal=True, prefix=True,
                 cap=20.0, culled=0.2), f"many {dim}")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("causal", [False, True])
def test_many_scenes_masks(device, dtype, bias, cap, causal):
    _check(_case(device, dtype, [300, 129] + MANY, 2, 1, 64, bias=bias, causal=causal, cap=cap,
                 culled=0.4), "masks")
    _check(_case(device, dtype, [70, 9, 130] + MANY, 2, 2, 64, bias=bias, causal=causal, cap=cap,
                 key_lengths=[200, 1, 40] + MANY), "other keys")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_many_scenes_masked_keys_reach_nothing(device, dtype, junk):
    c = _case(device, dtype, [150, 60] + MANY, 2, 2, 64, bias=True, culled=0.3, cap=8.0,
              key_lengths=[90, 171] + MANY)
    want = _run(c)
    for n in ("k", "v", "k_positions"):
        c[n] = c[n].clone()
        c[n][c["keep"] == 0] = junk
    got = _run(c)
    for n in got:
        assert torch.equal(got[n], want[n]), n
    for longest in (1, 100, 400):
        got = _run(c, longest=longest)
        for n in got:
            assert torch.equal(got[n], want[n]), (longest, n)


@pytest.mark.parametrize("kv", [28, 14, 4], ids=lambda k: f"kv{k}")
@pytest.mark.parametrize("dim,causal,cap,culled", [(64, False, 0.0, 0.1), (32, True, 9.0, 0.0)])
def test_long_scene_of_many_heads(device, kv, dim, causal, cap, culled):
    """Two heads of a wave share their distances, with one key head or two."""
    c = _case(device, BF16, [4100], 28, kv, dim, bias=True, causal=causal, cap=cap, culled=culled)
    _check(c, "pairs")
    got, want = _run(c, train=False)["out"], _run(c)["out"]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dim", [8, 40, 64, 128])
@pytest.mark.parametrize("cap", [0.0, 50.0])
@pytest.mark.parametrize("lengths", [[1, 1], [1] * 200], ids=["few", "many"])
def test_rows_that_see_one_key(device, dtype, dim, cap, lengths):
    """Their output is the key's value, and no gradient passes through their one weight: exactly."""
    c = _case(device, dtype, lengths, 4, 2, dim, bias=True, causal=True, cap=cap)
    got = _run(c)
    assert torch.equal(got["out"], c["v"].repeat_interleave(2, 1))
    for n in ("dq", "dk", "dslopes"):
        assert not got[n].any(), n
    R.assert_within(got["dv"], *(x["dv"] for x in R.attention(**c)), "dv")


# The results' rounding to bfloat16 is at most 2^-9 of each value.  Weights, ds and out enter the products
# with 16 bits: 2^-17 of each term, times what cancels in ds (2^4 here), times three.
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (50.0, True)])
@pytest.mark.parametrize("lengths", [[2] * 9, [3, 1, 2, 0, 5], [14, 4, 5], [2, 3] * 40], ids=str)
def test_few_keys_average_no_rounding(device, dim, cap, bias, lengths):
    """The gradients of tiny scenes are as exact as their own type."""
    c = _case(device, BF16, lengths, 4, 2, dim, bias=bias, causal=True, cap=cap)
    got = _run(c)
    want = R.attention(**c)[0]
    for n in ("out", "dq", "dk", "dv"):
        w = want[n].double()
        assert (got[n].double() - w).norm() <= (2.0 ** -9 + 2.0 ** -11) * w.norm(), n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("dim", [40, 64, 128])
@pytest.mark.parametrize("cap", [0.0, 50.0])
@pytest.mark.parametrize("lengths", [[70, 33], [900] * 16], ids=["few", "many"])
def test_first_causal_rows(device, dtype, dim, cap, lengths):
    """A causal scene's first row sees its own key alone, whatever its tile's other rows see."""
    c = _case(device, dtype, lengths, 4, 2, dim, bias=True, causal=True, cap=cap)
    got, first = _run(c), torch.tensor([sum(lengths[:n]) for n in range(len(lengths))], device=device)
    assert torch.equal(got["out"][first], c["v"][first].repeat_interleave(2, 1))
    assert not got["dq"][first].any()
