"""The operators on packed tokens: views, batches and routes that the operators' own files leave out."""
import pytest
import torch

import test_gpu_gated_norm as norms
import token_reference as R
from token_rounding import SLOPES, assert_rounded_once, assert_rounded_twice, off
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


# ---- scenes of few keys: two parts of bfloat16 carry the weights and ds, whatever the batch holds


def _case(device, dtype, lengths, H, K, D, key_lengths=None, bias=True, causal=False, cap=0.0, seed=0,
          offset=0.0, spread=40.0):
    g = _gen(device, seed)
    T, N = sum(lengths), sum(key_lengths or lengths)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=device).to(dtype)

    def starts(ls):
        return torch.tensor([0] + ls, device=device).cumsum(0).int()

    c = dict(q=normal(T, H, D), k=normal(N, K, D), v=normal(N, K, D), dout=normal(T, H, D),
             q_starts=starts(lengths), k_starts=starts(key_lengths) if key_lengths else None,
             causal=causal, cap=cap)
    if bias:
        c["q_positions"] = offset + spread * torch.rand(T, 3, generator=g, device=device)
        c["k_positions"] = (offset + spread * torch.rand(N, 3, generator=g, device=device)
                            if key_lengths else c["q_positions"])
        c["slopes"] = torch.tensor([2.0 ** -(h + 1) for h in range(H)], device=device).to(dtype)
    return c


def _run(c, **more):
    names = [n for n in ("q", "k", "v", "slopes") if n in c]
    v = {n: c[n].detach().clone().requires_grad_() for n in names}
    out = attention.scene_attention(
        v["q"], v["k"], v["v"], scene_starts=c["q_starts"], key_starts=c["k_starts"],
        causal=c["causal"], prefix=c.get("prefix"), cap=c["cap"], positions=c.get("q_positions"),
        key_positions=c.get("k_positions"), slopes=v.get("slopes"), keep=c.get("keep"), **more)
    got = torch.autograd.grad(out, list(v.values()), c["dout"])
    return {"out": out.detach(), **{"d" + n: g for n, g in zip(names, got)}}


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (50.0, True)])
@pytest.mark.parametrize("lengths,key_lengths", [
    ([2] * 64, None), ([2] * 65, None), ([2, 3] * 100, None), ([64] * 5, None), ([64] * 40, None),
    ([127, 1] * 30, None), ([200] * 2, [2] * 2), ([400] * 20, [3, 100] * 10)],
    ids=["2x64", "2x65", "2,3x100", "64x5", "64x40", "127,1x30", "200q2k", "400q3k"])
def test_scenes_of_few_keys_in_any_batch(device, dim, cap, bias, lengths, key_lengths):
    c = _case(device, BF16, lengths, 8, 2, dim, key_lengths=key_lengths, bias=bias, cap=cap)
    got, want = _run(c), R.attention(**c)[0]
    for n in ("out", "dq", "dk", "dv"):
        assert_rounded_once(got[n], want[n], n)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("others", [[], [5000], [300] * 30], ids=["alone", "long", "many"])
def test_a_short_scene_is_as_exact_beside_any_others(device, dim, others):
    c = _case(device, BF16, [2] * 9 + others, 8, 8, dim)
    got, want = _run(c), R.attention(**c)[0]
    for n in ("out", "dq", "dk", "dv"):
        assert_rounded_once(got[n][:18], want[n][:18], n)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (50.0, True)])
def test_short_caches(device, dim, cap, bias):
    """Caches of few live rows beside a long one; one row's value comes out as it is."""
    g, lengths, N = _gen(device, 3), [1, 2, 3, 9, 60, 127, 3000], 3000
    S, H, K = len(lengths), 8, 2
    q = torch.randn(S, H, dim, generator=g, device=device).to(BF16)
    k, v = (torch.randn(S, N, K, dim, generator=g, device=device).to(BF16) for _ in "kv")
    more = {}
    if bias:
        more = dict(positions=40 * torch.rand(S, 3, generator=g, device=device),
                    key_positions=40 * torch.rand(S, N, 3, generator=g, device=device),
                    slopes=torch.tensor([2.0 ** -(h + 1) for h in range(H)], device=device).to(BF16))
    got = attention.cached_attention(q, k, v, torch.tensor(lengths, dtype=torch.int32, device=device),
                                     cap=cap, **more)
    assert torch.equal(got[0], v[0, 0].repeat_interleave(H // K, 0))
    for s, n in enumerate(lengths[:-1]):
        ref = dict(q_positions=more["positions"][s:s + 1], k_positions=more["key_positions"][s, :n],
                   slopes=more["slopes"]) if bias else {}
        want = R.attention(q[s:s + 1], k[s, :n], v[s, :n], cap=cap, **ref)[0]["out"]
        assert_rounded_once(got[s:s + 1], want, n)


# ---- scenes are found from a workgroup's place


PACKINGS = {
    "long first": [2000] + [0] * 70 + [3] * 5 + [0] * 4000,
    "long last": [0] * 4000 + [3] * 5 + [0] * 70 + [2000],
    "far apart": ([0] * 99 + [40]) * 45,
    "among empty": [0] * 5 + [129] + [0] * 5,
    "even": [33] * 64,
    "even, one more": [33] * 65,
    "rising": list(range(0, 280, 4)),
}


@TYPES
@pytest.mark.parametrize("packing", PACKINGS)
@pytest.mark.parametrize("other_keys", [False, True], ids=["", "other keys"])
def test_packings(device, dtype, packing, other_keys):
    """Scenes of very different lengths, thousands of empty ones among them; with and without the longest
    scene's length, a wrong one too, the same bits."""
    lengths = PACKINGS[packing]
    keys = [(n + 5) // 2 if n else 0 for n in lengths] if other_keys else None
    c = _case(device, dtype, lengths, 2, 1, 32, key_lengths=keys, causal=True)
    got = _run(c)
    some = [n for n in lengths if n]
    near = dict(c, q_starts=_case(device, dtype, some, 2, 1, 32)["q_starts"])
    if keys:
        near["k_starts"] = _case(device, dtype, [n for n in keys if n], 2, 1, 32)["q_starts"]
    val, tol = R.attention(**near)  # a scene without rows has no part in the values
    for n in got:
        R.assert_within(got[n], val[n], tol[n], f"{packing} {n}")
    for longest in (1, max(lengths), sum(lengths)):
        again = _run(c, longest=longest)
        for n in got:
            assert torch.equal(again[n], got[n]), (longest, n)


@pytest.mark.parametrize("types", norms.TYPES, ids=["f32", "mixed", "bf16"])
@pytest.mark.parametrize("lengths", [
    [3] * 1500, [1] * 5000, [2000] + [0] * 70 + [1] * 1100 + [0] * 2000, [0] * 4000 + [2000], list(range(90)),
    [0] * 99 + [40] + [0] * 999 + [1]], ids=["3x1500", "1x5000", "long first", "long last", "rising", "far apart"])
def test_norm_packings(device, types, lengths):
    """Thousands of scenes: their gates and the sums over them; the longest scene's length changes nothing."""
    c = norms._case(device, sum(lengths), 40, lengths, types)
    got = norms._check(c)
    for longest in (1, max(lengths)):
        again = norms._run(c, longest=longest)
        for n in got:
            assert torch.equal(again[n], got[n]), (longest, n)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (50.0, True)])
def test_long_caches(device, dim, cap, bias):
    """Over long caches too the results are as exact as their type."""
    g, lengths, N = _gen(device, 5), [128, 129, 1000, 20_000], 20_000
    H, K = 32, 4
    q = torch.randn(4, H, dim, generator=g, device=device).to(BF16)
    k, v = (torch.randn(4, N, K, dim, generator=g, device=device).to(BF16) for _ in "kv")
    more = {}
    if bias:
        more = dict(positions=40 * torch.rand(4, 3, generator=g, device=device),
                    key_positions=40 * torch.rand(4, N, 3, generator=g, device=device),
                    slopes=torch.full((H,), 0.1, device=device).to(BF16))
    got = attention.cached_attention(q, k, v, torch.tensor(lengths, dtype=torch.int32, device=device),
                                     cap=cap, **more)
    for s, n in enumerate(lengths):
        ref = dict(q_positions=more["positions"][s:s + 1], k_positions=more["key_positions"][s, :n],
                   slopes=more["slopes"]) if bias else {}
        want = R.attention(q[s:s + 1], k[s, :n], v[s, :n], cap=cap, **ref)[0]["out"]
        assert_rounded_once(got[s:s + 1], want, n)


# ---- caps far above the scores


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("cap", [1000.0, 1e4, 1e5, 1e6])
@pytest.mark.parametrize("lengths", [[300], [300] + [140] * 90], ids=["few", "many"])
def test_large_caps(device, dim, bias, cap, lengths):
    """The nearer a cap is to none, the nearer its results are to those without one."""
    c = _case(device, BF16, lengths, 2, 2, dim, bias=bias, cap=cap)
    got, want = _run(c), R.attention(**c)[0]
    for n in ("out", "dq", "dk", "dv"):
        assert_rounded_twice(got[n], want[n], n)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("cap", [1000.0, 1e5, 1e6])
def test_large_caps_over_a_cache(device, dim, cap):
    g = _gen(device, 4)
    q = torch.randn(30, 8, dim, generator=g, device=device).to(BF16)
    k, v = (torch.randn(30, 400, 2, dim, generator=g, device=device).to(BF16) for _ in "kv")
    got = attention.cached_attention(q, k, v, torch.full((30,), 400, dtype=torch.int32, device=device), cap=cap)
    want = torch.cat([R.attention(q[s:s + 1], k[s], v[s], cap=cap)[0]["out"] for s in range(30)])
    assert_rounded_twice(got, want, "out")


# ---- what out in two parts and the rows' rests are for


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("cap", [0.0, 50.0])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,heads", [([450, 130], (2, 2)), ([450] * 8, (8, 2))], ids=["few", "many"])
def test_scores_with_clear_winners(device, dim, cap, causal, lengths, heads):
    """Rows with most of their weight on a few keys: the gradients are small differences, and within the bounds
    only with D from the whole output and the slopes' without the rows' rests (test_tokens_cpu.py)."""
    c = _case(device, BF16, lengths, *heads, dim, causal=causal, cap=cap, spread=256.0)
    c["q"], c["slopes"] = c["q"] * 4, c["slopes"].float() / 2
    got, want = _run(c), R.attention(**c)[0]
    for n in ("out", "dq", "dk", "dv"):
        assert_rounded_twice(got[n], want[n], n)
    assert off(got["dslopes"], want["dslopes"]) <= SLOPES


@TYPES
@pytest.mark.parametrize("offset", [1e5, 1e6])
@pytest.mark.parametrize("lengths", [[300], [300] + [1] * 200], ids=["few", "many"])
def test_positions_far_from_the_origin(device, dtype, offset, lengths):
    """Differences of positions come out of sums of bfloat16 products of the coordinates' parts: no less
    exact where the coordinates are large and the differences small."""
    c = _case(device, dtype, lengths, 2, 2, 64, offset=offset)
    got, (val, tol) = _run(c), R.attention(**c)
    for n in got:
        R.assert_within(got[n], val[n], tol[n], n)
    if dtype == BF16:
        assert_rounded_twice(got["out"][:300], val["out"][:300], "out")


# ---- which route a call takes, and captured training steps


@pytest.fixture
def taken(monkeypatch):
    """The native functions' answers, in order: whether each took its call."""
    assert _native.available
    log = []
    for name in ("rotate", "gated_norm", "scene_attention", "cached_attention"):
        def record(*args, call=getattr(_native, name)):
            out = call(*args)
            log.append(bool(out))
            return out
        monkeypatch.setattr(_native, name, record)
    return log


@TYPES
def test_plain_calls_take_the_native_nodes(device, taken, dtype):
    g = _gen(device, 6)

    def normal(*shape, t=dtype):
        return torch.randn(shape, generator=g, device=device).to(t)

    qkv = normal(50, 8, 48).requires_grad_()
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    pos = torch.rand(50, 4, generator=g, device=device)
    starts = torch.tensor([0, 20, 50], dtype=torch.int32, device=device)
    f = rotary.axis_frequencies((8, 8, 8), device=device)
    for interleaved in (False, True):
        rotary.rotate_qk(q, k, pos[:, :3], f, interleaved=interleaved)
    with torch.no_grad():
        rotary.rotate_qk(q, k, pos[:, :3], f)
    slopes = torch.rand(4, device=device)
    hits = torch.ones(50, dtype=torch.int32, device=device)
    for more in (dict(), dict(scene_starts=starts, longest=30), dict(causal=True, cap=5.0),
                 dict(scene_starts=starts, causal=True, prefix=starts[:2]), dict(scale=0.3),
                 dict(positions=pos[:, :3], slopes=slopes), dict(keep=hits), dict(keep=hits.bool()),
                 dict(positions=pos[:, :3], slopes=slopes.to(dtype), keep=hits.to(torch.uint8)),
                 dict(scene_starts=starts, key_starts=starts, positions=pos[:, :3], key_positions=pos[:, 1:],
                      slopes=slopes)):
        attention.scene_attention(q, k, v, **more)
        with torch.no_grad():
            attention.scene_attention(q, k, v, **more)
    with torch.no_grad():
        n = torch.tensor([50], dtype=torch.int32, device=device)
        attention.cached_attention(q[:1], k[None], v[None], n)
        attention.cached_attention(q[:1], k[None], v[None], n, cap=5.0, positions=pos[:1, :3],
                                   key_positions=pos[None, :, :3], slopes=slopes, keep=hits[None])
    x, w = normal(50, 40, t=F32).requires_grad_(), torch.rand(40, device=device)
    for stream, branch in ((x, normal(50, 40)), (normal(50, 40), normal(50, 40))):
        for more in (dict(), dict(scale=w, branch_weight=w), dict(gate=normal(50, 40)), dict(gate=normal(1, 40)),
                     dict(gate=normal(2, 40), scene_starts=starts, longest=30), dict(gate=normal(1, 40, t=F32))):
            gated_norm.gated_residual_norm(stream, branch, w, **more)
    assert taken == [True] * len(taken) and len(taken) == 3 + 20 + 2 + 12


@TYPES
def test_calls_the_native_nodes_leave(device, taken, dtype):
    """Empty batches, rows off alignment, strided last axes: the Python classes do them, and give the values
    of plain tensors."""
    g = _gen(device, 7)
    q = torch.randn(30, 2, 32, generator=g, device=device).to(dtype)
    want = attention.scene_attention(q, q, q)
    odd = torch.zeros(30, 2, 33, dtype=dtype, device=device)[..., 1:].copy_(q)
    strided = q.transpose(1, 2).contiguous().transpose(1, 2)
    for t in (odd, strided):
        assert torch.equal(attention.scene_attention(t, q, t), want)
    assert attention.scene_attention(q[:0], q[:0], q[:0]).shape == (0, 2, 32)
    f, pos = torch.rand(1, 16, device=device), torch.rand(30, 1, device=device)
    rotary.rotate_qk(q, None, pos, f)  # not asked
    rotary.rotate_qk(strided, q, pos, f)
    w = torch.ones(32, device=device)
    gated_norm.gated_residual_norm(strided[:, 0], q[:, 0], w)
    gated_norm.gated_residual_norm(q[:0, 0], q[:0, 0], w)
    assert taken == [True] + [False] * 6


@pytest.mark.parametrize("scenes", [[40, 33, 1], [5] * 200], ids=["few", "many"])
def test_a_captured_training_step(device, route, scenes):
    """A block of all three operators with their gradients in a HIP graph: each replay, after new
    inputs and eager work, equals the eager step."""
    g, T, H, D = _gen(device, 8), sum(scenes), 4, 32
    C = H * D

    def normal(*shape):
        return torch.randn(shape, generator=g, device=device).to(BF16)

    starts = torch.tensor([0] + scenes, device=device).cumsum(0).int()
    pos, f = 40 * torch.rand(T, 3, generator=g, device=device), rotary.axis_frequencies((6, 5, 5), device=device)
    w = torch.rand(C, generator=g, device=device)
    inputs = [normal(T, 3 * H, D), normal(T, C), normal(len(scenes), C), torch.full((H,), 0.1, device=device)]
    grads = normal(T, C), normal(T, C)

    def step():
        # (views as leaves: nothing but these operators' kernels is captured)
        qkv, x, gate, slopes = inputs
        leaves = [t.detach().requires_grad_() for t in (qkv[:, :H], qkv[:, H:2 * H], qkv[:, 2 * H:], x, gate, slopes)]
        q, k = rotary.rotate_qk(*leaves[:2], pos, f)
        o = attention.scene_attention(q, k, leaves[2], scene_starts=starts, causal=True, cap=20.0,
                                      positions=pos, slopes=leaves[5])
        out = gated_norm.gated_residual_norm(leaves[3], o.flatten(1), w, branch_weight=w, gate=leaves[4],
                                             scene_starts=starts)
        return out + torch.autograd.grad(out, leaves, grads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(4):
        for t in inputs[:3]:
            t.copy_(torch.randn(t.shape, generator=g, device=device))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), n


# ---- traces, modes and transforms


@pytest.fixture(params=["rotary", "norm", "attention", "attention with grad", "cached"])
def operator(request, device):
    """(a call of one operator on a (6, 4, 32) tensor, that tensor)."""
    g = _gen(device, 9)
    pos, f = torch.rand(6, 3, generator=g, device=device), rotary.axis_frequencies((6, 5, 5), device=device)
    w, cache = torch.rand(32, device=device), torch.randn(6, 9, 2, 32, generator=g, device=device)
    n = torch.tensor([0, 1, 5, 9, 9, 3], dtype=torch.int32, device=device)
    starts = torch.tensor([0, 2, 6], dtype=torch.int32, device=device)
    slopes = torch.rand(4, generator=g, device=device)

    def scene(q):
        return attention.scene_attention(q, q[:, :2], q[:, 2:], scene_starts=starts, causal=True, cap=9.0,
                                         positions=pos, slopes=slopes)

    call = {"rotary": lambda q: rotary.rotate_qk(q, q[:, :2], pos, f)[1],
            "norm": lambda q: gated_norm.gated_residual_norm(q[:, 0], q[:, 1], w, scale=w, gate=q[:2, 2],
                                                             scene_starts=starts)[1],
            "attention": scene, "attention with grad": scene,
            "cached": lambda q: attention.cached_attention(q, cache, cache, n)}[request.param]
    q = torch.randn(6, 4, 32, generator=g, device=device)
    return call, q.requires_grad_(request.param == "attention with grad")


def test_a_trace_replays_on_other_values(operator, request):
    """A traced call is recorded with its checks: other inputs give their own results; a count of tokens that
    the other tensors do not have is refused before anything is launched, and one that they allow (the
    norm's starts end with the rows) is taken."""
    call, q = operator
    traced = torch.jit.trace(call, (q,))
    for n in range(3):
        x = (q.detach() * (n + 2)).requires_grad_(q.requires_grad)
        assert torch.equal(traced(x), call(x)), n
    x = q.detach()[:5].contiguous().requires_grad_(q.requires_grad)
    if request.node.callspec.params["operator"] == "norm":
        assert torch.equal(traced(x), call(x))
    else:
        with pytest.raises(RuntimeError, match="ValueError|must|need"):
            traced(x)


def test_modes_and_transforms(operator):
    """Dispatch and function modes change nothing; what has no rule here raises, and loses nothing silently."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    class Functions(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    call, q = operator
    want = call(q)
    for mode in (Dispatch, Functions):
        with mode():
            assert torch.equal(call(q), want), mode
    x = q.detach()
    with forward_ad.dual_level():
        assert torch.equal(call(x), want)  # no tangent: nothing to lose
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(forward_ad.make_dual(x, x))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.vmap(call)(torch.stack((x, x)))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(call, (x,), (x,))
    with FakeTensorMode(allow_non_fake_inputs=True) as mode, pytest.raises(RuntimeError):
        call(mode.from_tensor(x))


# ---- long scenes, through the kernels of large calls, elementwise


def _within(c, what):
    got, (val, tol) = _run(c), R.attention(**c)
    for n in got:
        R.assert_within(got[n], val[n], tol[n], f"{what} {n}")
    return got


@TYPES
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("causal,cap,bias", [(False, 0.0, True), (True, 30.0, True), (True, 0.0, False)])
def test_long_scenes(device, dtype, dim, causal, cap, bias):
    c = _case(device, dtype, [2600, 900], 8, 2, dim, causal=causal, cap=cap, bias=bias)
    if causal:
        c["prefix"] = torch.tensor([600, 0], dtype=torch.int32, device=device)
    c["keep"] = torch.rand(3500, generator=_gen(device, 1), device=device) >= 0.05
    _within(c, "long")


@pytest.mark.parametrize("kv", [8, 4, 1], ids=lambda k: f"kv{k}")
@pytest.mark.parametrize("dim,cap", [(32, 9.0), (64, 9.0), (64, 0.0)])
def test_pairs_of_heads_over_several_scenes(device, kv, dim, cap):
    """Two heads of a wave share their distances, also where no scene alone would fill the chip; the results
    of a training call and of one without gradients are the same bits."""
    c = _case(device, BF16, [2000, 511, 2300, 1500], 24, 3 * kv, dim, cap=cap)
    c["keep"] = torch.rand(6311, generator=_gen(device, 1), device=device) >= 0.05
    got = _within(c, "pairs")
    with torch.no_grad():
        again = attention.scene_attention(
            c["q"], c["k"], c["v"], scene_starts=c["q_starts"], cap=cap, positions=c["q_positions"],
            slopes=c["slopes"], keep=c["keep"])
    assert torch.equal(again, got["out"])


# ---- launches past a grid's x axis


@pytest.mark.parametrize("longest", [None, 1], ids=["by tiles", "by slots"])
@pytest.mark.parametrize("first", [1, 5000], ids=["even", "long first"])
def test_hundreds_of_thousands_of_scenes(device, first, longest):
    """More workgroups than the grid's x axis takes (four million), scenes looked for over three levels: a
    token alone in its scene has its own value, and its gradient goes there."""
    n, H, D = 300_000, 16, 8
    starts = torch.cat((torch.zeros(1, device=device), first + torch.arange(n, device=device))).int()
    T, g = n + first - 1, _gen(device, 10)
    q, k, v, dout = (torch.randn(T, H, D, generator=g, device=device).to(BF16) for _ in range(4))
    slopes = torch.full((H,), 0.1, device=device)
    pos = torch.rand(T, 3, generator=g, device=device)
    leaves = [t.requires_grad_() for t in (q, k, v, slopes)]
    out = attention.scene_attention(*leaves[:3], scene_starts=starts, longest=longest, positions=pos,
                                    slopes=leaves[3])
    got = torch.autograd.grad(out, leaves, dout)
    alone = slice(first if first > 1 else 0, None)
    assert torch.equal(out[alone], v[alone]) and torch.equal(got[2][alone], dout[alone])
    assert not got[0][alone].any() and not got[1][alone].any()
    if first > 1:
        one = attention.scene_attention(q[:first], k[:first], v[:first], positions=pos[:first], slopes=leaves[3])
        assert off(out[:first], one.detach().double()) <= 2.0 ** -8
    else:
        assert not got[3].any()


def test_norm_of_more_scenes_than_a_grid_s_axis(device):
    norms._check(norms._case(device, 66_000, 8, [1] * 66_000, (F32, BF16)))
