"""The optimiser's step on a GPU against its formulas in 64 bits."""
import copy
import pickle

import pytest
import torch

import token_reference as R
from gs_voxelizer import _native, adamw

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


@pytest.fixture(params=["native", "python"])
def route(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_native, "available", False)
    else:
        assert _native.available
    return request.param


KINDS = {"f32": (F32, F32, False), "f32, bf16 grad": (F32, BF16, False), "bf16": (BF16, BF16, False),
         "bf16, f32 grad": (BF16, F32, False), "masters": (BF16, BF16, True), "masters, f32 grad": (BF16, F32, True)}


class Step:
    """Tensors of given shapes and kinds, in the middle of a training."""

    def __init__(self, device, shapes, kinds, seed=0, offset=0, grad_scale=1e-3):
        g = torch.Generator(device=device).manual_seed(seed)

        def normal(shape, scale, dtype):
            n = 1
            for x in shape:
                n *= x
            x = torch.zeros(n + offset, dtype=dtype, device=device)
            x[offset:] = (scale * torch.randn(n, generator=g, device=device)).to(dtype)
            return x[offset:].view(shape)

        self.params, self.grads, self.exp_avgs, self.exp_avg_sqs, self.masters = [], [], [], [], []
        for shape, kind in zip(shapes, kinds):
            p_type, g_type, master = KINDS[kind]
            w = normal(shape, 0.05, F32)
            self.params.append(normal(shape, 0.0, p_type).copy_(w))
            self.masters.append(w if master else None)
            self.grads.append(normal(shape, grad_scale, g_type))
            self.exp_avgs.append(normal(shape, 5e-4, F32))
            self.exp_avg_sqs.append(normal(shape, 1e-3, F32).square_())

    def run(self, step=7, **more):
        return adamw.adamw_step(self.params, self.grads, self.exp_avgs, self.exp_avg_sqs, step,
                                **dict(dict(masters=self.masters), **more))

    def check(self, step=7, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, max_norm=None, count=None):
        """One step, within what 32-bit arithmetic may be off: 1 - beta, beta and the rates are rounded once, each
        product and sum once; a quotient adds its operands' relative errors, a root halves its own."""
        before = [[None if t is None else t.double().clone() for t in ts] for ts in
                  (self.params, self.masters, self.grads, self.exp_avgs, self.exp_avg_sqs)]
        n = len(self.params)
        norm = self.run(step, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, max_norm=max_norm)
        total = sum(float((g ** 2).sum()) for g in before[2]) ** 0.5
        by = 1.0
        if max_norm is None:
            assert norm is None
        else:
            assert norm.shape == () and norm.dtype == F32
            assert abs(float(norm) - total) <= 2 * U * total
            by = min(1.0, max_norm / (total + 1e-6))
        b1, b2 = betas
        for i in range(n):
            p, w, g, m, v = (x[i] for x in before)
            t = count if count is not None else step[i] if isinstance(step, list) else step
            rate = lr[i] if isinstance(lr, (list, tuple)) else lr
            rate = float(rate)
            decay = weight_decay[i] if isinstance(weight_decay, (list, tuple)) else weight_decay
            g = g * by
            m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
            tm = 1.01 * U * (3 * (b1 * m).abs() + 6 * ((1 - b1) * g).abs()) + 1e-44
            tv = 1.01 * U * (3 * b2 * v + 9 * (1 - b2) * g ** 2) + 1e-44
            den = (v1 / (1 - b2 ** t)).sqrt() + eps
            up = rate / (1 - b1 ** t) * m1 / den
            old = p if w is None else w
            new = old * (1 - rate * decay) - up
            # sqrt(v1 + tv) - sqrt(v1) is at most sqrt(tv)
            root = torch.minimum(tv / (2 * v1.sqrt()).clamp_min(1e-300), tv.sqrt()) / (1 - b2 ** t) ** 0.5
            tw = 1.01 * (U * 3 * old.abs() + up.abs() * (root / den + 10 * U)
                         + rate / (1 - b1 ** t) * tm / den) + 1e-44
            R.assert_within(self.exp_avgs[i], m1, tm, f"exp_avg {i}")
            R.assert_within(self.exp_avg_sqs[i], v1, tv, f"exp_avg_sq {i}")
            if w is not None:
                R.assert_within(self.masters[i], new, tw, f"master {i}")
                assert torch.equal(self.params[i], self.masters[i].to(BF16)), i
            elif p.numel():
                u = 0 if self.params[i].dtype == F32 else 2.0 ** -8
                R.assert_within(self.params[i], new, tw + u * (new.abs() + tw), f"param {i}")
        return norm


SIZES = [1, 2, 3, 4, 5, 255, 1023, 1024, 1025, 4099, 100_003]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("max_norm", [None, 0.1], ids=["", "clipped"])
def test_sizes(device, route, kind, max_norm):
    s = Step(device, [(n,) for n in SIZES] + [(0,), (7, 11, 13), ()], [kind] * (len(SIZES) + 3))
    s.check(weight_decay=0.1, max_norm=max_norm)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_off_alignment(device, kind, offset):
    """Views that begin anywhere in a buffer: the same bits as aligned ones."""
    shapes = [(n,) for n in SIZES]
    a, b = (Step(device, shapes, [kind] * len(shapes), offset=o) for o in (0, offset))
    for c in (a, b):
        c.check(max_norm=0.05)
    for x, y in zip(a.params + a.exp_avgs + a.exp_avg_sqs, b.params + b.exp_avgs + b.exp_avg_sqs):
        assert torch.equal(x, y)


@pytest.mark.parametrize("max_norm", [None, 1e-2, 1e6], ids=["", "clipped", "not clipped"])
@pytest.mark.parametrize("counted", [False, True], ids=["host", "device"])
def test_many_tensors_of_all_kinds(device, route, max_norm, counted):
    """More than a launch's table holds, of each kind, with a rate, decay and step of their own."""
    n = 300
    kinds = [list(KINDS)[i * 7 % 6] for i in range(n)]
    s = Step(device, [(1 + (i * 37) % 200, 1 + i % 5) for i in range(n)], kinds)
    rates, decays = [1e-4 * (1 + i % 9) for i in range(n)], [0.03 * (i % 4) for i in range(n)]
    if counted:
        counter = torch.tensor([4], dtype=torch.int32, device=device)
        s.check(counter, lr=rates, weight_decay=decays, max_norm=max_norm, count=5)
        assert counter.tolist() == [5]
    else:
        s.check([1 + i % 50 for i in range(n)], lr=rates, weight_decay=decays, max_norm=max_norm)


@pytest.mark.parametrize("kind", KINDS)
def test_large_tensors(device, kind):
    """Past 8 million elements a workgroup takes 4,096; a first step, with odd sizes beside it."""
    s = Step(device, [(3001, 3001), (5,), (4097,), (12_289,)], [kind] * 4)
    for ts in (s.exp_avgs, s.exp_avg_sqs):
        for t in ts:
            t.zero_()
    s.check(1, max_norm=0.5, weight_decay=0.01)


@pytest.mark.parametrize("betas,eps,step", [((0.0, 0.0), 1e-8, 1), ((0.9, 0.999), 0.0, 3), ((0.95, 0.9999), 1e-15, 1),
                                            ((0.5, 0.99), 1.0, 10 ** 6), ((0.9, 0.999), 1e-8, 2 ** 31)])
def test_constants(device, route, betas, eps, step):
    s = Step(device, [(5000,), (33,)], ["f32", "masters"])
    s.check(step, betas=betas, eps=eps, lr=0.1, weight_decay=0.5)


def test_gradients_of_zero_and_far_values(device, route):
    """Nothing moves where there is no gradient and no state (0 / eps), and squares past float32's range are the
    formula's infinity; the norm is summed past it."""
    s = Step(device, [(1000,), (1000,)], ["f32", "masters"])
    for ts in (s.grads, s.exp_avgs, s.exp_avg_sqs):
        for t in ts:
            t.zero_()
    before = [t.clone() for t in s.params]
    s.run(1, lr=0.1)
    assert all(torch.equal(a, b) for a, b in zip(before, s.params))
    s = Step(device, [(1000,), (7,)], ["f32", "f32"], grad_scale=1.0)
    s.grads[0].fill_(1e30)
    norm = s.check(3, max_norm=1.0)
    assert abs(float(norm) / (1e30 * 1000 ** 0.5) - 1) < 1e-6
    s = Step(device, [(1000,), (7,)], ["f32", "f32"], grad_scale=1.0)
    s.exp_avgs[1].zero_(), s.exp_avg_sqs[1].zero_()
    s.grads[0].fill_(1e30)
    s.run(3)
    assert torch.isinf(s.exp_avg_sqs[0]).all() and torch.isfinite(s.params[0]).all()
    assert torch.isfinite(s.params[1]).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_gradient_that_is_not_finite(device, route, bad):
    """Without max_norm it reaches its own element alone; with it, as torch's clip_grad_norm_ has it."""
    s, c = (Step(device, [(1000,), (50,)], ["f32", "f32"]) for _ in "ab")
    for x in (s, c):
        x.grads[0][7] = bad
    s.run()
    assert torch.isfinite(s.params[0]).sum() == 999 and torch.isfinite(s.params[1]).all()
    norm = c.run(max_norm=1.0)
    assert not torch.isfinite(norm)
    want = [torch.nn.Parameter(t.clone()) for t in c.grads]
    for w in want:
        w.grad = w.detach().clone()
    torch.nn.utils.clip_grad_norm_(want, 1.0)
    for w, m in zip(want, c.exp_avgs):
        assert torch.equal(torch.isnan(w.grad), torch.isnan(m))


def test_layouts(device, route):
    """Dense tensors in any order of their axes; a gradient laid out otherwise is taken as if alike."""
    a, b, c = (Step(device, [(40, 3, 5)], ["f32"]) for _ in "abc")
    a.check()
    for s in (b, c):
        for n in ("params", "exp_avgs", "exp_avg_sqs"):
            t = getattr(s, n)[0]
            getattr(s, n)[0] = t.permute(2, 0, 1).contiguous().permute(1, 2, 0)
            assert not getattr(s, n)[0].is_contiguous()
    c.grads[0] = torch.cat((c.grads[0], c.grads[0]), 2)[..., :5]
    for s in (b, c):
        s.run()
        for n in ("params", "exp_avgs", "exp_avg_sqs"):
            assert torch.equal(getattr(s, n)[0], getattr(a, n)[0])


def test_rates_on_the_device(device, route):
    rates = [torch.tensor(3e-3, device=device), 1e-3, torch.tensor([5e-2], device=device)]
    s = Step(device, [(1000,), (99,), (5000,)], ["f32", "masters", "bf16"])
    s.check(lr=rates, weight_decay=[0.1, 0.2, 0.3])
    s.check(lr=rates[0], max_norm=0.1)


def test_a_gradient_of_two_parameters(device, route):
    s = Step(device, [(100,), (100,)], ["f32", "f32"])
    s.grads[1] = s.grads[0]
    s.check(max_norm=0.001)


def test_runs_repeat(device):
    a, b = (Step(device, [(100_000,), (3000, 1000), (17,)], ["f32", "masters", "bf16"]) for _ in "ab")
    for step in range(1, 6):
        assert torch.equal(a.run(step, max_norm=0.5), b.run(step, max_norm=0.5))
    for n in ("params", "exp_avgs", "exp_avg_sqs"):
        assert all(torch.equal(x, y) for x, y in zip(getattr(a, n), getattr(b, n)))


def test_captured_steps(device, route):
    """A step in a graph counts on, clips by the gradients it finds and reads the rate it finds."""
    shapes, kinds = [(5000,), (33, 7), (257,)], ["f32", "masters", "bf16"]
    a, b = (Step(device, shapes, kinds) for _ in "ab")
    counters = [torch.zeros(1, dtype=torch.int32, device=device) for _ in "ab"]
    rate = torch.tensor(1e-3, device=device)
    more = dict(lr=rate, weight_decay=0.1, max_norm=0.05)
    for s, c in zip((a, b), counters):
        s.run(c, **more)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = a.run(counters[0], **more)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="count on the device"):
            a.run(3)
        a.grads[0].add_(0)  # (a graph of its own, with something in it)
    g = torch.Generator(device=device).manual_seed(3)
    for i in range(6):
        for x, y in zip(a.grads, b.grads):
            x.copy_(10.0 ** -(i % 5) * torch.randn(x.shape, generator=g, device=device))
            y.copy_(x)
        rate.fill_(1e-3 * (i + 1))
        graph.replay()
        want = b.run(counters[1], **more)
        assert torch.equal(norm, want) and torch.equal(*counters) and int(counters[0]) == i + 2
        for n in ("params", "exp_avgs", "exp_avg_sqs"):
            assert all(torch.equal(x, y) for x, y in zip(getattr(a, n), getattr(b, n))), (i, n)
        assert torch.equal(a.masters[1], b.masters[1])
        torch.cuda.synchronize()


def test_streams(device):
    """Steps of two sets of tensors on two streams at once."""
    a, b, c, d = (Step(device, [(200_000,), (77,)], ["f32", "masters"], seed=i // 2) for i in range(4))
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for step in range(1, 8):
        for s, stream in zip((a, c), streams):
            with torch.cuda.stream(stream):
                s.run(step, max_norm=0.1)
    torch.cuda.synchronize()
    for step in range(1, 8):
        b.run(step, max_norm=0.1), d.run(step, max_norm=0.1)
    for x, y in ((a, b), (c, d)):
        for n in ("params", "exp_avgs", "exp_avg_sqs"):
            assert all(torch.equal(p, q) for p, q in zip(getattr(x, n), getattr(y, n)))


def test_autograd_sees_the_writes(device, route):
    s = Step(device, [(50,)], ["f32"])
    w = torch.ones(50, device=device, requires_grad=True)
    loss = (s.params[0] * w).sum()
    s.run()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        Step(device, [(50,)], ["f32"]).run()


def test_refusals(device):
    s = Step(device, [(50,), (20,)], ["f32", "bf16"])
    before = [t.clone() for t in s.params + s.exp_avgs]

    def no(text, **more):
        a = dict(params=s.params, grads=s.grads, exp_avgs=s.exp_avgs, exp_avg_sqs=s.exp_avg_sqs, step=1)
        with pytest.raises(ValueError, match=text):
            adamw.adamw_step(**dict(a, **more))

    f, h = s.params
    no("hold a tensor", params=[], grads=[], exp_avgs=[], exp_avg_sqs=[])
    no("grads must hold 2", grads=s.grads[:1])
    no("masters must hold 2", masters=[None])
    no("CUDA tensor", params=[f.cpu(), h])
    no("CUDA tensor", params=[f.double(), h])
    no("gaps", params=[torch.zeros(100, device=device)[::2], h])
    no("shape and device", grads=[s.grads[0][:49], s.grads[1]])
    no("shape and device", grads=[s.grads[0].double(), s.grads[1]])
    no("shape and device", exp_avgs=[s.exp_avgs[0].to(BF16), s.exp_avgs[1]])
    no("laid out like", params=[torch.zeros(5, 10, device=device).t()], grads=[torch.zeros(10, 5, device=device)],
       exp_avgs=[torch.zeros(10, 5, device=device)], exp_avg_sqs=[torch.zeros(10, 5, device=device)])
    no("needs none", masters=[torch.zeros(50, device=device), None])
    no("shares memory", exp_avgs=[s.exp_avgs[0], s.exp_avgs[0][:20]])
    no("shares memory", grads=[f, s.grads[1]])
    no("shares memory", grads=[s.grads[0], s.exp_avg_sqs[0][30:]])
    no("whole numbers", step=2**64 + 1)
    no("shares memory", params=[f, f], grads=[s.grads[0]] * 2, exp_avgs=[s.exp_avgs[0], f.clone()],
       exp_avg_sqs=[s.exp_avg_sqs[0], f.clone()])
    no("whole numbers", step=0)
    no("whole numbers", step=1.5)
    no("step must be one value or 2", step=[1])
    no("int32", step=torch.ones(1, device=device))
    no("int32", step=torch.ones(1, dtype=torch.int32))
    no("lr must not be negative", lr=-1.0)
    no("lr must be numbers", lr="1")
    no("lr must be one value or 2", lr=[1e-3])
    no("one element", lr=torch.ones(2, device=device))
    no("one element", lr=torch.ones(1))
    no("weight_decay must not", weight_decay=-0.1)
    no("betas", betas=(1.0, 0.9))
    no("eps", eps=-1.0)
    no("max_norm", max_norm=0.0)
    no("max_norm", max_norm=-1.0)
    for a, b in zip(s.params + s.exp_avgs, before):
        assert torch.equal(a, b)


# ---- the optimiser


def _model(device, dtype=F32, seed=0):
    torch.manual_seed(seed)
    m = torch.nn.Sequential(torch.nn.Linear(6, 33), torch.nn.GELU(), torch.nn.Linear(33, 5, bias=False))
    return m.to(device=device, dtype=dtype)


def _grads(m, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    for p in m.parameters():
        p.grad = torch.randn(p.shape, generator=g, device=p.device).to(p.dtype)


def _groups(m):
    ps = list(m.parameters())
    return [dict(params=ps[:1], weight_decay=0.3), dict(params=ps[1:], lr=5e-3)]


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_as_torch_s_in_64_bits(device, capturable, max_norm):
    """Ten steps with groups, a changing rate and clipping, beside torch's optimiser in float64.  Each step adds what
    32 bits are off in an update, 2^-20 of the rate at most, and a rounding of the weight."""
    m = _model(device)
    d = copy.deepcopy(m).double()
    opt = adamw.AdamW(_groups(m), lr=1e-3, weight_decay=0.1, max_norm=max_norm, capturable=capturable)
    ref = torch.optim.AdamW(_groups(d), lr=1e-3, weight_decay=0.1)
    for i in range(10):
        _grads(m, i)
        for p, q in zip(m.parameters(), d.parameters()):
            q.grad = p.grad.double()
        norm = torch.nn.utils.clip_grad_norm_(d.parameters(), max_norm) if max_norm else None
        for o in (opt, ref):
            o.param_groups[1]["lr"] = 5e-3 / (i + 1)
            o.step()
        if max_norm:
            assert abs(float(opt.norm) / float(norm) - 1) < 2.0 ** -22
    for p, q in zip(m.parameters(), d.parameters()):
        assert float((p - q).detach().abs().max()) <= 10 * (2.0 ** -20 * 5e-3 + 2.0 ** -24 * float(q.detach().abs().max()))


def test_masters_keep_small_updates(device):
    """Updates below half a bfloat16 spacing, step by step: lost without masters, kept with them."""
    ends = []
    for masters in (False, True):
        p = torch.nn.Parameter(torch.ones(100, dtype=BF16, device=device))
        opt = adamw.AdamW([p], lr=1e-4, weight_decay=0.0, masters=masters)
        for _ in range(100):
            p.grad = torch.ones_like(p)
            opt.step()
        ends.append(p.detach().clone())
    assert (ends[0] == 1).all()
    assert (ends[1].float() - 0.99).abs().max() <= 2.0 ** -8 * 0.99


@pytest.mark.parametrize("masters", [False, True])
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_state_is_saved_and_loaded(device, masters, capturable, dtype, tmp_path):
    """A run that is saved, loaded and run on gives the bits of one that was not; the state stays float32."""
    def steps(m, opt, which):
        for i in which:
            _grads(m, i)
            opt.step()

    def new(m):
        return adamw.AdamW(_groups(m), lr=1e-2, masters=masters, max_norm=1.0, capturable=capturable)

    m = _model(device, dtype)
    opt = new(m)
    steps(m, opt, range(3))
    torch.save((m.state_dict(), opt.state_dict()), tmp_path / "run.pt")
    pickled = pickle.dumps(opt)
    steps(m, opt, range(3, 6))
    again = _model(device, dtype, seed=1)
    model_state, opt_state = torch.load(tmp_path / "run.pt", weights_only=True)
    again.load_state_dict(model_state)
    other = new(again)
    other.load_state_dict(opt_state)
    for s in other.state.values():
        assert all(t.dtype == F32 for n, t in s.items() if n != "step")
        assert ("master" in s) == (masters and dtype == BF16)
    steps(again, other, range(3, 6))
    for p, q in zip(m.parameters(), again.parameters()):
        assert torch.equal(p, q)
    loaded = pickle.loads(pickled)
    assert (loaded.masters, loaded.max_norm, loaded.capturable) == (masters, 1.0, capturable)


def test_parameters_without_a_gradient(device):
    """They are left alone, and count only their own steps."""
    a, b = (torch.nn.Parameter(torch.ones(10, device=device)) for _ in "ab")
    opt = adamw.AdamW([a, b], lr=1e-2)
    opt.step()
    assert not opt.state
    for i in range(4):
        a.grad, b.grad = torch.ones_like(a), torch.ones_like(b) if i % 2 else None
        opt.step()
    assert opt.state[a]["step"] == 4 and opt.state[b]["step"] == 2
    assert (b > a).all() and (b < 1).all()


def test_closure_and_scheduler(device):
    p = torch.nn.Parameter(torch.ones(10, device=device))
    opt = adamw.AdamW([p], lr=1e-2)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, 0.1)

    def closure():
        opt.zero_grad()
        loss = (p ** 2).sum()
        loss.backward()
        return loss

    assert float(opt.step(closure).detach()) == 10
    sched.step()
    assert abs(opt.param_groups[0]["lr"] - 1e-3) < 1e-12


def test_captured_optimiser(device):
    """The whole step of a fit in two graphs: gradients, then the optimiser; as eager steps, to the bit."""
    target = torch.linspace(0, 1, 300, device=device).view(100, 3)
    runs = []
    for captured in (False, True):
        p = torch.nn.Parameter(torch.zeros(100, 3, device=device))
        opt = adamw.AdamW([p], lr=1e-2, capturable=True, max_norm=1.0)

        def backward():
            p.grad = None
            ((p - target) ** 2).sum().backward()

        backward()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            with pytest.raises(RuntimeError, match="before the capture"):
                opt.step()
            target.add(0)
        opt.step()
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                backward()
            torch.cuda.current_stream().wait_stream(side)
            first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
            with torch.cuda.graph(first):
                backward()
            with torch.cuda.graph(second):
                opt.step()
        for _ in range(5):
            if captured:
                first.replay(), second.replay()
            else:
                backward(), opt.step()
            torch.cuda.synchronize()
        runs.append(p.detach().clone())
        assert int(opt.state[p]["step"]) == 6
    assert torch.equal(*runs)


def test_groups_that_are_refused(device):
    a, b = (torch.nn.Parameter(torch.ones(10, device=device)) for _ in "ab")
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    for more in (dict(max_norm=1.0), dict(capturable=True)):
        opt = adamw.AdamW([dict(params=[a]), dict(params=[b], betas=(0.5, 0.9))], **more)
        with pytest.raises(ValueError, match="betas"):
            opt.step()
    adamw.AdamW([dict(params=[a]), dict(params=[b], betas=(0.5, 0.9))]).step()
    for more in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1), dict(weight_decay=-1), dict(max_norm=0)):
        with pytest.raises(ValueError):
            adamw.AdamW([a], **more)


def test_a_captured_fit_of_gaussians(device):
    """A fit through the voxelizer in two graphs: a replay's step is the formula's on the gradients that it left."""
    from gs_voxelizer import graph, synthetic, voxelize
    from helpers import small_config
    from test_gpu_graph import _make
    voxelize._capacity.pop(device.index or 0, None)
    leaves, backward = _make(device, small_config(1, 3000, vol=(48, 40, 56)), seed=3)
    rates = [1e-4, 2e-4, 1e-3, 1e-2]
    opt = adamw.AdamW([dict(params=[p], lr=r) for p, r in zip(leaves, rates)], weight_decay=0.0, capturable=True)
    voxelize_and_differentiate = graph.CapturedStep(backward)
    opt.step()
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        opt.step()
    for i in range(4):
        voxelize_and_differentiate.replay()
        before = [[t.detach().double().clone() for t in (p, p.grad, opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq"])]
                  for p in leaves]
        second.replay()
        torch.cuda.synchronize()
        t = i + 2
        for p, r, (w, g, m, v) in zip(leaves, rates, before):
            m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
            up = r * (m / (1 - 0.9 ** t)) / ((v / (1 - 0.999 ** t)).sqrt() + 1e-8)
            # an update is at most r / (1 - 0.9) here, and 2^-20 of that off; the weight rounds once
            assert float((p.detach() - (w - up)).abs().max()) <= 2.0 ** -20 * 10 * r + 2.0 ** -23 * float(w.abs().max())
    assert int(opt.state[leaves[0]]["step"]) == 5


def test_plain_calls_take_the_native_step(device, monkeypatch):
    assert _native.available
    log = []
    call = _native.adamw_step

    def record(*args):
        out = call(*args)
        log.append(out[0])
        return out

    monkeypatch.setattr(_native, "adamw_step", record)
    s = Step(device, [(50,), (3, 4)], ["f32", "masters"])
    counter = torch.zeros(1, dtype=torch.int32, device=device)
    for step in (3, [3, 4], counter):
        for more in (dict(), dict(max_norm=1.0), dict(lr=[1e-3, 1e-2], weight_decay=(0.1, 0)), dict(lr=1)):
            s.run(step, **more)
    p = torch.nn.Parameter(torch.ones(5, device=device))
    p.grad = torch.ones_like(p)
    adamw.AdamW([p]).step()
    adamw.AdamW([p], capturable=True, max_norm=1.0).step()
    assert len(log) == 14 and all(log)
    s.run(lr=torch.tensor(1e-3, device=device))
    assert not log[-1]


@pytest.mark.parametrize("count", [1, 8, 9, 32, 33, 44, 45, 88, 160, 161, 321])
@pytest.mark.parametrize("empty", [False, True], ids=["", "with empty ones"])
def test_as_many_tensors_as_a_launch_takes(device, count, empty):
    """Launches take so many tensors each: the last one full, or with one more to come."""
    shapes, kinds = [(1 + (i * 613) % 1500,) for i in range(count)], ["f32"] * count
    if empty:
        shapes, kinds = [(0,)] + shapes[:count // 2] + [(0,)] + shapes[count // 2:], kinds + ["bf16", "f32"]
    s = Step(device, shapes, kinds)
    counter = torch.tensor([2], dtype=torch.int32, device=device)
    s.check(counter, weight_decay=0.1, max_norm=0.02, count=3)
    assert counter.tolist() == [3]
    s = Step(device, shapes, kinds)
    s.check(weight_decay=0.1)
