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


# ---- which rows are read, exactly
#
# Scores are 0 or so low that their weight is 0 in binary32, and values are small whole numbers: a result is the mean of
# the values of the rows that count, sum and number exact, divided and rounded.  A row that is left out, read twice
# or taken from another page shows, however many there are.


def _waves_and_keys(dtype, dim):
    return (2 if dim > 64 else 4), (32 if dtype == BF16 else 16)


def _workgroups(dtype, heads, kv_heads, dim):
    """Workgroups of a key head and 16 of its query heads, as the launch cuts a batch (one round of them)."""
    waves, keys = _waves_and_keys(dtype, dim)
    wide = 32 if dim <= 32 else 64 if dim <= 64 else 128
    lds = waves * (4 * keys * wide * (2 if dtype == BF16 else 4) + 6 * keys * 4) + 2048
    return 256 * min(163840 // lds, 4) // (kv_heads * -(-heads // kv_heads // 16))


class Chosen:
    """A cache whose rows count or do not, for each query head by one channel of its keys, by the positions (bias) and by
    a mask (keep); what no call may look at is NaN.  gone: the share of the table's entries that name no page."""

    def __init__(self, device, dtype, lengths, H, K, D, rows=48, cap=0.0, bias=False, keep=False, gone=0.0, seed=0):
        g = _gen(device, seed)
        S, self.rows, self.cap = len(lengths), rows, cap
        n = _ints(lengths, device).long()
        need = -(-n // rows)
        P, most = int(need.sum()) + 3, max(int(need.max()), 1)
        order = torch.randperm(P, generator=g, device=device)
        place = torch.arange(most, device=device)
        used = place < need[:, None]
        first = need.cumsum(0) - need
        table = order[(first[:, None] + place).clamp(max=P - 1)]
        live = torch.zeros(P, rows, dtype=torch.bool, device=device)
        at = torch.arange(rows, device=device)
        live[table[used]] = (place[:, None] * rows + at < n[:, None, None])[used]
        self.scene_of = torch.zeros(P, dtype=torch.long, device=device)
        self.scene_of[table[used]] = torch.arange(S, device=device)[:, None].expand(S, most)[used]

        def flips(*shape, share):
            return torch.rand(shape, generator=g, device=device) < share

        self.values = torch.randint(-8, 9, (P, rows, K, D), generator=g, device=device, dtype=torch.int8)
        self.chosen = flips(P, rows, K, D, share=0.3)
        nan = torch.tensor(float("nan"), dtype=dtype, device=device)
        self.keep = flips(P, rows, share=0.5) if keep else None
        seen = live if self.keep is None else live & self.keep
        self.counts = seen
        k = torch.where(self.chosen, 0.0, -64.0).to(dtype)
        self.k_pages = torch.where(seen[..., None, None], k, nan)
        self.v_pages = torch.where(seen[..., None, None], self.values.to(dtype), nan)
        self.channel = torch.randint(0, D, (S, H), generator=g, device=device)
        self.q = torch.zeros(S, H, D, dtype=dtype, device=device).scatter_(2, self.channel[..., None], 64.0)
        self.positions = self.position_pages = self.slopes = None
        if bias:
            self.positions = 100 * torch.rand(S, 3, generator=g, device=device)
            near = flips(P, rows, share=0.4)
            here = self.positions[self.scene_of][:, None].expand(P, rows, 3)
            self.position_pages = torch.where(near[..., None], here, here + 3000.0)
            self.position_pages[~live] = float("nan")
            self.slopes = torch.tensor([2.0 ** -(h % 3) for h in range(H)], device=device).to(dtype)
            self.counts = seen & near
        self.there = used & ~flips(S, most, share=gone)
        bad = _ints([-1, -(2**31), 2**31 - 1, P], device).long()
        bad = bad[torch.randint(0, 4, (S, most), generator=g, device=device)]
        self.pages, self.table = table, torch.where(self.there, table, bad).int()
        self.lengths = n.int()

    def run(self):
        return paged.paged_attention(self.q, self.k_pages, self.v_pages, self.table, self.lengths, cap=self.cap,
                                     positions=self.positions, position_pages=self.position_pages, slopes=self.slopes,
                                     keep_pages=self.keep)

    def check(self, heads=None):
        got = self.run()
        S, H, D = got.shape
        group, told = H // self.k_pages.shape[2], 0
        for s in range(S):
            pages = self.pages[s][self.there[s]]
            seen = self.counts[pages]
            for h in range(H) if heads is None else heads:
                c = int(self.channel[s, h])
                rows = seen & self.chosen[pages, :, h // group, c]
                number = int(rows.sum())
                if not number:  # whether keys of other channels are seen then decides: only told where none is
                    if not int((self.keep[pages] & self._live(s, pages) if self.keep is not None
                                else self._live(s, pages)).sum()):
                        assert not got[s, h].any(), (s, h)
                    continue
                total = (self.values[pages, :, h // group] * rows[..., None]).sum((0, 1), dtype=torch.int64)
                mean = total.double() / number
                ends = [(mean * x).to(got.dtype) for x in (1 - 2.0 ** -23, 1 + 2.0 ** -23)]  # the quotient's rounding
                low, high = torch.minimum(*ends), torch.maximum(*ends)
                assert ((low <= got[s, h]) & (got[s, h] <= high)).all(), (s, h, number)
                told += 1
        assert torch.equal(got, self.run())
        return told

    def _live(self, s, pages):
        i = torch.nonzero(self.there[s])
        return i * self.rows + torch.arange(self.rows, device=i.device) < int(self.lengths[s])


OPTIONS = pytest.mark.parametrize("options", [dict(), dict(bias=True, keep=True, gone=0.1), dict(cap=1e3, gone=0.1)],
                                  ids=["plain", "bias, mask, gaps", "cap, gaps"])


@TYPES
@pytest.mark.parametrize("dim,kv_heads", [(8, 32), (64, 16), (128, 16)])
@OPTIONS
def test_many_steps_of_a_wave_in_pieces(device, dtype, dim, kv_heads, options):
    """A wave reads its pages' numbers 32 steps at a time, 16 ahead: here it takes 70 and more, with gaps everywhere."""
    waves, keys = _waves_and_keys(dtype, dim)
    shares = _workgroups(dtype, kv_heads, kv_heads, dim)
    rows = (shares - 1) * 70 * waves * keys + 1037
    c = Chosen(device, dtype, [rows], kv_heads, kv_heads, dim, **options)
    assert 2 < shares and rows // (shares * waves * keys) > 64
    assert c.check(heads=range(0, kv_heads, 5)) > 0


@TYPES
@pytest.mark.parametrize("dim,kv_heads", [(8, 64), (64, 32), (128, 64)])
@OPTIONS
def test_many_steps_of_a_wave_in_shares(device, dtype, dim, kv_heads, options):
    """Likewise in equal shares, that end and begin inside scenes, with empty and short ones between."""
    waves, keys = _waves_and_keys(dtype, dim)
    shares = _workgroups(dtype, kv_heads, kv_heads, dim)
    each = 72 * waves * keys  # a share's rows
    lengths = [5, int(1.7 * each), 0, int(2.31 * each), 33, 0, 1, int(1.2 * each) + 7]
    lengths += [17] * max(0, (shares + 1) // 2 - len(lengths))
    lengths.append(shares * each - sum(lengths))
    assert 2 * len(lengths) >= shares and lengths[-1] > each
    c = Chosen(device, dtype, lengths, kv_heads, kv_heads, dim, **options)
    assert c.check(heads=range(1, kv_heads, 9)) > 0


@TYPES
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("cap", [0.0, 1e3, 1e4])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("keep,gone", [(False, 0.0), (True, 0.15)], ids=["", "mask, gaps"])
def test_every_variant_in_equal_shares(device, dtype, dim, cap, bias, keep, gone):
    """Scenes of all lengths, so that a workgroup ends one and goes on in the next."""
    lengths = [(311 * s * s + 7 * s) % 900 * (s % 5 > 0) for s in range(70)]
    assert 2 * len(lengths) >= _workgroups(dtype, 8, 8, dim)
    c = Chosen(device, dtype, lengths, 8, 8, dim, cap=cap, bias=bias, keep=keep, gone=gone)
    assert c.check(heads=(0, 3, 7)) > 100


@TYPES
@pytest.mark.parametrize("heads,kv_heads,dim", [(128, 4, 64), (68, 4, 40), (96, 3, 128), (256, 8, 32)])
def test_more_heads_than_a_workgroup_takes_in_equal_shares(device, dtype, heads, kv_heads, dim):
    lengths = [(311 * s * s + 7 * s) % 700 * (s % 7 > 0) for s in range(70)]
    assert 2 * len(lengths) >= _workgroups(dtype, heads, kv_heads, dim)
    c = Chosen(device, dtype, lengths, heads, kv_heads, dim, bias=True, keep=True, gone=0.1)
    assert c.check(heads=(0, 15, 16, 17, heads // kv_heads - 1, heads // kv_heads, heads - 1)) > 100


@TYPES
@pytest.mark.parametrize("scenes", [1000, 5000])
def test_thousands_of_scenes(device, dtype, scenes):
    """A lane looks at many scenes where it cuts the batch."""
    lengths = [(97 * s) % 70 * (s % 4 > 0) for s in range(scenes)]
    for s in (0, scenes // 3, scenes - 1):
        lengths[s] = 3001 + s % 7
    c = Chosen(device, dtype, lengths, 2, 1, 32, rows=16, bias=True, gone=0.05)
    assert c.check(heads=(1,)) > scenes // 2


@TYPES
def test_values_in_equal_shares(device, dtype):
    """Ordinary scores and values there, against the formula."""
    lengths = [(311 * s * s + 7 * s) % 300 * (s % 5 > 0) for s in range(70)]
    for cap, bias, keep in ((0.0, False, 0.0), (0.0, True, 0.4), (30.0, False, 0.0), (2e3, True, 0.0)):
        c = Case(device, dtype, lengths, 16, 8, 64, rows=48, cap=cap, bias=bias, keep=keep)
        assert 2 * len(lengths) >= _workgroups(dtype, 16, 8, 64)
        c.check(c.run(), scenes=range(0, 70, 6))


@TYPES
def test_a_prompt_that_continues_a_cache(device, dtype):
    """Appended at once; its tokens attend in one call as scenes that share their pages, each with a row more."""
    g, H, K, D, rows, old, new = _gen(device, 6), 4, 2, 64, 16, 37, 30
    T = old + new
    x = torch.randn(T, H + 2 * K, D, generator=g, device=device).to(dtype)
    pool = torch.full((7, 2, rows, K, D), float("nan"), dtype=dtype, device=device)
    cache = pool[:, 0], pool[:, 1]
    table = _ints([[4, 0, 6, 2, 5]], device)
    for first, last in ((0, old), (old, T)):
        paged.append_tokens(x[first:last, H:H + K], x[first:last, H + K:], *cache, table, _ints([last], device),
                            scene_starts=_ints([0, last - first], device))
    lengths = torch.arange(old + 1, T + 1, dtype=torch.int32, device=device)
    got = paged.paged_attention(x[old:, :H], *cache, table.expand(new, -1), lengths)
    val, tol = R.attention(x[old:, :H], x[:, H:H + K], x[:, H + K:], causal=True)  # the last rows of the scene's
    R.assert_within(got, val["out"], tol["out"], "continued")
