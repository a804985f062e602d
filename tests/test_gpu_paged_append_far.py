"""Appending to batches of as many scenes as there may be."""
import pytest
import torch

from gs_voxelizer import _tokens, paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("boundary", [2048, 2050, 2051])
@pytest.mark.parametrize("scenes", [2**30 + 5, _tokens.MAX_TOKENS])
def test_scenes_that_lie_far_apart(device, scenes, boundary):
    """Tokens of one workgroup in the second scene and in the one before the last, with more than 2^30 empty ones
    between; they share a table's row, and write different rows of it."""
    T, D, rows = 4096, 8, 16
    g = torch.Generator(device=device).manual_seed(1)
    k, v = (torch.randn(T, 1, D, generator=g, device=device) for _ in "kv")
    pools = [torch.zeros(T // rows, rows, 1, D, device=device) for _ in "kv"]
    order = torch.randperm(T // rows, generator=g, device=device).int()
    starts = torch.full((scenes + 1,), boundary, dtype=torch.int32, device=device)
    starts[:2] = 0
    starts[scenes - 1:] = T
    lengths = torch.zeros(scenes, dtype=torch.int32, device=device)
    lengths[1], lengths[scenes - 2] = boundary, T
    paged.append_tokens(k, v, *pools, order[None].expand(scenes, -1), lengths, scene_starts=starts)
    for got, want in zip(pools, (k, v)):
        assert torch.equal(got[order.long()].flatten(0, 1), want)
