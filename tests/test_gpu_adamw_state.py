"""Steps that are counted for each tensor on its own, and the optimiser's state as it is made and loaded."""
import copy

import pytest
import torch

from gs_voxelizer import _native, adamw
from test_gpu_adamw import BF16, F32, KINDS, U, Step

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"])
def route(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_native, "available", False)
    else:
        assert _native.available
    return request.param


class Counted(Step):
    """Step i of `check` is counted by counters[i] (a number: by the host)."""

    def run(self, step=7, **more):
        return super().run(self.counters, **more)


def _counters(device, counts):
    return [torch.tensor([n - 1], dtype=torch.int32, device=device) for n in counts]


@pytest.mark.parametrize("max_norm", [None, 0.02], ids=["", "clipped"])
@pytest.mark.parametrize("n", [1, 4, 28, 257, 600])
def test_a_counter_for_each(device, route, max_norm, n):
    """As many as a launch counts and more, of all kinds, an empty tensor among them."""
    kinds = [list(KINDS)[i * 7 % 6] for i in range(n)]
    s = Counted(device, [(1 + (i * 613) % 1500,) if i != 2 else (0,) for i in range(n)], kinds)
    counts = [1 + (i * 37) % 1000 for i in range(n)]
    order = [(i * 5) % n for i in range(n)] if n % 5 else list(range(n))
    made = _counters(device, [counts[i] for i in order])  # not in memory's order
    s.counters = [made[order.index(i)] for i in range(n)]
    for _ in range(2):
        s.check(counts, weight_decay=0.1, max_norm=max_norm)
        assert [int(c) for c in s.counters] == counts
        counts = [c + 1 for c in counts]


def test_counters_that_tensors_share_and_numbers_among_them(device, route):
    s = Counted(device, [(100,), (2000,), (7,), (300,), (1025,)], ["f32", "masters", "bf16", "f32", "f32"])
    a, b = _counters(device, [5, 90])
    s.counters = [a, b, 3, b, a]
    s.check([5, 90, 3, 90, 5], max_norm=0.1)
    assert (int(a), int(b)) == (5, 90)
    s.counters = [a, b, 4, b, a]
    s.check([6, 91, 4, 91, 6])
    assert (int(a), int(b)) == (6, 91)


def test_large_tensors_with_counters(device):
    """Workgroups of 4,096 elements, and more sums of squares than the update's workgroups add up."""
    s = Counted(device, [(3001, 3001), (5,), (12_289,)], ["masters", "f32", "bf16, f32 grad"])
    s.counters = _counters(device, [2, 70, 1])
    s.check([2, 70, 1], max_norm=0.5)


def test_counters_that_are_refused(device, route):
    s = Step(device, [(50,), (20,)], ["f32", "bf16"])
    c = torch.ones(1, dtype=torch.int32, device=device)
    for bad in (c.float(), c.cpu(), torch.ones(2, dtype=torch.int32, device=device), c[0], c.long()):
        with pytest.raises(ValueError, match="int32"):
            s.run([c, bad])
    with pytest.raises(ValueError, match="one value or 2"):
        s.run([c])
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="count on the device"):
            s.run([c, 3])
        s.grads[0].add_(0)
    assert int(c) == 1


def test_autograd_sees_the_counts(device, route):
    s = Step(device, [(50,), (20,)], ["f32", "masters"])
    cs = _counters(device, [3, 4])
    before = [t._version for t in cs + s.params + s.exp_avgs + s.exp_avg_sqs + s.masters[1:]], [g._version for g in s.grads]
    s.run(cs)
    after = [t._version for t in cs + s.params + s.exp_avgs + s.exp_avg_sqs + s.masters[1:]], [g._version for g in s.grads]
    assert all(a > b for a, b in zip(after[0], before[0])) and after[1] == before[1]


# ---- the optimiser


def _grad(shape, g, device):
    """Gradients of one sign, from 0.5 to 1.5: their moments' roundings do not cancel."""
    return 0.5 + torch.rand(shape, generator=g, device=device)


def _near(ps, ds, rate, steps):
    """Beside torch's optimiser in float64.  A moment is off by 3 (the first) or 4 (the second) roundings of 2^-24 a
    step, relatively, the root halves the second's; 8 more come with the update, which is at most 3 rates, as
    gradients differ by a factor of 3; and the weight rounds 3 times a step."""
    for p, d in zip(ps, ds):
        one = 3 * rate * U * (3 * steps + 2 * steps + 8) + 3 * U * float(d.detach().abs().max())
        assert float((p.double() - d).detach().abs().max()) <= 1.01 * steps * one


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("max_norm", [None, 2.0])
@pytest.mark.parametrize("order", ["late", "skips", "both"])
def test_gradients_that_come_late_or_not_always(device, capturable, max_norm, order):
    """Each parameter's updates are corrected for the steps that it made."""
    g = torch.Generator(device=device).manual_seed(1)
    ps = [torch.nn.Parameter(torch.rand(n, generator=g, device=device)) for n in (100, 30, 1500)]
    ds = [torch.nn.Parameter(p.detach().double()) for p in ps]
    opt = adamw.AdamW(ps, lr=1e-2, weight_decay=0.1, capturable=capturable, max_norm=max_norm)
    ref = torch.optim.AdamW(ds, lr=1e-2, weight_decay=0.1)
    steps = [0, 0, 0]
    for i in range(12):
        has = [True, i >= 5 if order != "skips" else True, i % 3 > 0 if order != "late" else True]
        for k, (p, d) in enumerate(zip(ps, ds)):
            p.grad = _grad(p.shape, g, device) if has[k] else None
            d.grad = p.grad.double() if has[k] else None
            steps[k] += has[k]
        if max_norm:
            torch.nn.utils.clip_grad_norm_(ds, max_norm)
        opt.step(), ref.step()
    assert [int(opt.state[p]["step"]) for p in ps] == steps
    _near(ps, ds, 1e-2, 12)


@pytest.mark.parametrize("capturable", [False, True])
def test_loaded_counts_that_differ(device, capturable):
    """torch's state after 1,000 steps of one parameter and 1 of another goes on as torch goes on."""
    g = torch.Generator(device=device).manual_seed(2)
    ps = [torch.nn.Parameter(torch.rand(n, generator=g, device=device)) for n in (64, 65)]
    ds = [torch.nn.Parameter(p.detach().double()) for p in ps]
    ref = torch.optim.AdamW(ds, lr=1e-2)
    for d, n in zip(ds, (1000, 1)):
        x = _grad(d.shape, g, device).double()
        by = [1 - b ** n for b in (0.9, 0.999)]  # as n steps with this gradient leave it, rounded to 32 bits
        ref.state[d] = dict(step=torch.tensor(float(n)), exp_avg=(by[0] * x).float().double(),
                            exp_avg_sq=(by[1] * x * x).float().double())
    opt = adamw.AdamW(ps, lr=1e-2, capturable=capturable)
    opt.load_state_dict(copy.deepcopy(ref.state_dict()))
    for i in range(3):
        for p, d in zip(ps, ds):
            p.grad = _grad(p.shape, g, device)
            d.grad = p.grad.double()
        opt.step(), ref.step()
    assert [int(opt.state[p]["step"]) for p in ps] == [1003, 4]
    _near(ps, ds, 1e-2, 3)


def test_replays_count_what_they_step(device):
    """Graphs of a step of two parameters and of one, and eager steps between: each replay counts its own parameters,
    to the bit as eager steps do."""
    g = torch.Generator(device=device).manual_seed(3)
    runs = []
    first = [torch.rand(n, generator=g, device=device) for n in (100, 1500)]
    grads = [_grad(t.shape, g, device) for t in first]
    for captured in (False, True):
        ps = [torch.nn.Parameter(t.clone()) for t in first]
        opt = adamw.AdamW(ps, lr=1e-2, capturable=True, max_norm=1.0)

        def step(both):
            for p, x, on in zip(ps, grads, (True, both)):
                p.grad = x if on else None
            opt.step()

        step(True)
        graphs = {}
        if captured:
            for both in (True, False):
                graphs[both] = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graphs[both]):
                    step(both)
        for i, both in enumerate([True, False, False, True, True, False, True, True]):
            if captured and i != 4:
                graphs[both].replay()
            else:
                step(both)
            torch.cuda.synchronize()
        runs.append([p.detach().clone() for p in ps])
        assert [int(opt.state[p]["step"]) for p in ps] == [9, 6]
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_looking_at_the_state_changes_nothing(device):
    """The state of a parameter that was looked at before its first step is made all the same."""
    for capturable in (False, True):
        ps = [torch.nn.Parameter(torch.ones(5, device=device)) for _ in "ab"]
        opt = adamw.AdamW(ps, capturable=capturable)
        assert not opt.state[ps[0]] and not opt.state[ps[1]]
        ps[0].grad = torch.ones_like(ps[0])
        opt.step()
        assert int(opt.state[ps[0]]["step"]) == 1 and not opt.state[ps[1]]


@pytest.mark.parametrize("capturable", [False, True])
def test_masters_on_off_and_on_again(device, capturable):
    """A checkpoint with masters goes on without them, and later with new ones: no step brings old weights back."""
    def run(masters, state=None, weights=None, dtype=BF16, steps=40):
        p = torch.nn.Parameter(torch.ones(100, dtype=dtype, device=device))
        if weights is not None:
            p.data.copy_(weights)
        opt = adamw.AdamW([p], lr=1e-2, weight_decay=0.0, masters=masters, capturable=capturable)
        if state is not None:
            opt.load_state_dict(state)
        for _ in range(steps):
            p.grad = torch.ones_like(p)
            opt.step()
        return p.detach().clone(), copy.deepcopy(opt.state_dict())

    on, on_state = run(True)
    off, off_state = run(False, on_state, on)
    assert "master" not in off_state["state"][0]
    again, _ = run(True, off_state, off, steps=1)
    # constant gradients: each step is the rate but for 1e-4 of it, and a bfloat16 of this size rounds by 2^-9 at most
    assert (off < on - 0.3).all()
    assert ((again.float() - (off.float() - 1e-2)).abs() <= 1e-6 + 2.0 ** -9).all()
    wide, wide_state = run(True, on_state, on.float(), dtype=F32, steps=1)
    assert "master" not in wide_state["state"][0]
    assert ((wide - (on.float() - 1e-2)).abs() <= 2e-6).all()
