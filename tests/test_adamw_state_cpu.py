"""The optimiser's state without a GPU: what is loaded, and what the C entry makes of counters."""
import ctypes

import pytest
import torch

from gs_voxelizer import _lib, adamw

OK, INVALID = 0, 1


def _loaded(counts, capturable):
    """An optimiser that has loaded torch's state of parameters with these step counts."""
    ps = [torch.nn.Parameter(torch.ones(3)) for _ in counts]
    ref = torch.optim.AdamW([torch.nn.Parameter(torch.ones(3)) for _ in counts], lr=1e-2)
    for p, n in zip(ref.param_groups[0]["params"], counts):
        if n:
            ref.state[p] = dict(step=torch.tensor(float(n)), exp_avg=torch.full((3,), 0.5),
                                exp_avg_sq=torch.full((3,), 0.25))
    opt = adamw.AdamW(ps, lr=1e-2, capturable=capturable)
    opt.load_state_dict(ref.state_dict())
    return opt, ps


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("counts", [[1000, 1], [1, 1000, 7], [3, 0, 3]])
def test_each_parameter_keeps_its_count(capturable, counts):
    opt, ps = _loaded(counts, capturable)
    for p, n in zip(ps, counts):
        assert (int(opt.state[p]["step"]) == n) if n else p not in opt.state
    if capturable:
        steps = [opt.state[p]["step"] for p, n in zip(ps, counts) if n]
        assert all(t.dtype == torch.int32 and t.shape == (1,) for t in steps)
        steps[0] += 1  # what one's step counts, no other's does
        assert [int(t) for t in steps] == [n + (i == 0) for i, n in enumerate(n for n in counts if n)]
        again = adamw.AdamW(ps, lr=1e-2, capturable=True)
        again.load_state_dict(opt.state_dict())
        assert [int(again.state[p]["step"]) for p, n in zip(ps, counts) if n] == [int(t) for t in steps]


def _plan(counters, **more):
    tensors = [_lib.AdamwTensor(param=(1 << 20) + (i << 16), grad=(2 << 30) + (i << 16), exp_avg=(3 << 30) + (i << 16),
                                exp_avg_sq=(4 << 30) + (i << 16), numel=100, step=0 if c else 1, counter=c)
               for i, c in enumerate(counters)]
    all = (_lib.AdamwTensor * len(tensors))(*tensors)
    a = _lib.Adamw(tensors=ctypes.addressof(all), count=len(tensors), beta1=0.9, beta2=0.999, eps=1e-8, **more)
    n = ctypes.c_size_t(0)
    return _lib.load().gsv_adamw_workspace_bytes(ctypes.byref(a), ctypes.byref(n)), n.value


def test_counters_of_tensors():
    assert _plan([1024, None, 1028]) == (OK, 16)  # two corrections each
    assert _plan([1024, 1024, None], max_norm=1.0) == (OK, 3 * 8 + 2 * 8 + 16)
    assert _plan([1026])[0] == INVALID
    assert _plan([1024, None], counter=2048)[0] == INVALID


def _with_state(dtype, masters, master=None):
    p = torch.nn.Parameter(torch.full((3,), 5.0, dtype=dtype))
    opt = adamw.AdamW([p], masters=masters)
    opt.state[p] = dict(step=4, exp_avg=torch.full((3,), 0.5), exp_avg_sq=torch.full((3,), 0.25))
    if master is not None:
        opt.state[p]["master"] = torch.full((3,), master)
    return opt, p


@pytest.mark.parametrize("dtype,masters", [(torch.bfloat16, False), (torch.float32, True), (torch.float32, False)],
                         ids=["off", "float32", "float32, off"])
def test_masters_are_loaded_where_they_are_kept(dtype, masters):
    """Elsewhere they would only grow old: in the state, and in what is saved from it."""
    saved, _ = _with_state(torch.bfloat16, True, 5.0078125)
    opt, p = _with_state(dtype, masters)
    opt.load_state_dict(saved.state_dict())
    assert set(opt.state[p]) == {"step", "exp_avg", "exp_avg_sq"}
    # back on, with the weights as they are by then
    again, q = _with_state(torch.bfloat16, True)
    again.load_state_dict(opt.state_dict())
    assert again.state[q]["master"].tolist() == [5.0] * 3 and again.state[q]["master"].dtype == torch.float32
    same, q = _with_state(torch.bfloat16, True)
    same.load_state_dict(saved.state_dict())
    assert same.state[q]["master"].tolist() == [5.0078125] * 3


def test_states_that_are_refused():
    """Another optimiser's, or another model's: nothing is loaded."""
    def saved(make, shape=(3,), **more):
        p = torch.nn.Parameter(torch.ones(shape))
        p.grad = torch.ones_like(p)
        ref = make([p], **dict(dict(lr=0.5), **more))
        ref.step()
        return ref.state_dict()

    opt, p = _with_state(torch.float32, False)
    for state in (saved(torch.optim.AdamW, amsgrad=True), saved(torch.optim.AdamW, maximize=True),
                  saved(torch.optim.Adam, weight_decay=0.1), saved(torch.optim.SGD, momentum=0.9),
                  saved(torch.optim.RMSprop), saved(torch.optim.AdamW, (1,)), saved(torch.optim.AdamW, (2, 3))):
        with pytest.raises(ValueError):
            opt.load_state_dict(state)
        assert opt.state[p]["step"] == 4 and opt.param_groups[0]["lr"] == 1e-3
    other, _ = _with_state(torch.bfloat16, True, 1.0)
    state = other.state_dict()
    state["state"][0]["master"] = torch.ones(1)
    with pytest.raises(ValueError, match="master"):
        opt.load_state_dict(state)
    for state in (saved(torch.optim.AdamW), saved(torch.optim.AdamW, foreach=True), saved(torch.optim.Adam)):
        opt.load_state_dict(state)
        assert opt.state[p]["step"] == 1 and opt.param_groups[0]["lr"] == 0.5
        assert opt.state[p]["exp_avg"].tolist() == pytest.approx([0.1] * 3)


@pytest.mark.parametrize("capturable", [False, True])
def test_a_state_that_was_looked_at_and_is_empty(capturable):
    ps = [torch.nn.Parameter(torch.ones(3)) for _ in "ab"]
    opt = adamw.AdamW(ps, capturable=capturable)
    assert not opt.state[ps[0]]
    again = adamw.AdamW(ps, capturable=capturable)
    again.load_state_dict(opt.state_dict())
    assert not again.state[ps[0]] and not again.state[ps[1]]
