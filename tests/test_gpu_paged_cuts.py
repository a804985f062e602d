"""Attention over a cache in pages: how batches and scenes are cut, in many steps, equal shares and large batches."""
import pytest
import torch

import token_reference as R
from gs_voxelizer import paged
from test_gpu_paged import BF16, F32, TYPES, Case, _gen, _ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scenes,heads", [((1 << 19) - 1, 16), (1 << 19, 16), ((1 << 20) - 1, 16), ((1 << 21) - 3, 4)])
def test_batches_whose_rows_pass_a_grid_s_axis(device, scenes, heads):
    """2^23 rows of 16 heads and more, in a batch that is split: some long scenes, all others of a row or none."""
    g = _gen(device, 1)
    rows, D, most = 16, 8, 9
    k, v = (torch.randn(40, rows, 1, D, generator=g, device=device).to(BF16) for _ in "kv")
    q = torch.randn(scenes, heads, D, generator=g, device=device).to(BF16)
    lengths = (torch.arange(scenes, device=device) % 3 != 1).to(torch.int32)
    table = (torch.arange(scenes, device=device) % 40).int()[:, None].expand(-1, most).contiguous()
    long = {0: 144, 7: 130, scenes // 2: 144, scenes - 2: 97, scenes - 1: 143}
    for s, n in long.items():
        lengths[s] = n
        table[s] = _ints([(s + 7 * i) % 40 for i in range(most)], device)
    got = paged.paged_attention(q, k, v, table, lengths)
    one = lengths == 1
    want = v[table[:, 0].long(), 0].expand(-1, heads, -1)
    assert torch.equal(got[one], want[one]) and not got[lengths == 0].any()
    for s, n in long.items():
        at = [(int(table[s, j // rows]), j % rows) for j in range(n)]
        kk, vv = (torch.stack([t[p, r] for p, r in at]) for t in (k, v))
        val, tol = R.attention(q[s:s + 1], kk, vv)
        R.assert_within(got[s:s + 1], val["out"], tol["out"], s)
