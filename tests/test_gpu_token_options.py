"""What the attention operators take as scale and cap, on both routes."""
import pytest
import torch

from gs_voxelizer import _native, attention, paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("route", ["native", "python"])
@pytest.mark.parametrize("bad", [dict(cap=float("inf")), dict(cap=1e39), dict(scale=float("inf")), dict(scale=1e39),
                                 dict(cap=float("nan")), dict(scale=float("nan"))])
def test_infinities_are_refused(device, monkeypatch, route, bad):
    if route == "python":
        monkeypatch.setattr(_native, "available", False)
    x = torch.randn(16, 2, 64, device=device)
    cache, n = x.view(1, 16, 2, 64), torch.tensor([16], dtype=torch.int32, device=device)
    table = torch.zeros(1, 1, dtype=torch.int32, device=device)
    for call in (lambda **a: attention.scene_attention(x, x, x, **a),
                 lambda **a: attention.cached_attention(x[:1], cache, cache, n, **a),
                 lambda **a: paged.paged_attention(x[:1], cache, cache, table, n, **a)):
        with pytest.raises(ValueError, match="scale must be|cap must not"):
            call(**bad)
        assert torch.isfinite(call(cap=1e30)).all()
