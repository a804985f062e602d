"""The cache in pages on a GPU: tokens appended to it, and attention over it, against the formulas in 64 bits."""
import pytest
import torch

import token_reference as R
from token_rounding import assert_rounded_once, assert_rounded_twice
from gs_voxelizer import _native, attention, paged, rotary

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])


@pytest.fixture(params=["native", "python"])
def route(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_native, "available", False)
    else:
        assert _native.available
    return request.param


def _gen(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


class Case:
    """Scenes' rows, laid together and in pages handed out in no order.  What no scene's live row holds is NaN."""

    def __init__(self, device, dtype, lengths, H, K, D, rows=16, cap=0.0, bias=True, keep=0.0, joint=False, seed=0,
                 room=0, spread=40.0):
        g = _gen(device, seed)
        S, top = len(lengths), max(max(lengths), 1)
        self.lengths, self.cap, self.rows = lengths, cap, rows
        self.q = torch.randn(S, H, D, generator=g, device=device).to(dtype)
        self.k, self.v = (torch.randn(S, top, K, D, generator=g, device=device).to(dtype) for _ in "kv")
        need = [-(-n // rows) for n in lengths]
        P, most = sum(need) + 2, max(need) + room
        order = torch.randperm(P, generator=g, device=device).tolist()
        self.table = torch.full((S, max(most, 1)), -1, dtype=torch.int32, device=device)
        pool = torch.full((P, 2, rows, K, D), float("nan"), dtype=dtype, device=device)
        self.k_pages, self.v_pages = (pool[:, 0], pool[:, 1]) if joint else (pool[:, 0].clone(), pool[:, 1].clone())
        self.positions = self.key_positions = self.position_pages = self.slopes = None
        if bias:
            self.positions = spread * torch.rand(S, 3, generator=g, device=device)
            self.key_positions = spread * torch.rand(S, top, 3, generator=g, device=device)
            self.position_pages = torch.full((P, rows, 3), float("nan"), device=device)
            self.slopes = torch.tensor([2.0 ** -(h + 1) for h in range(H)], device=device).to(dtype)
        self.keep = self.keep_pages = None
        if keep:
            self.keep = (torch.rand(S, top, generator=g, device=device) >= keep).to(torch.int32) * 27
            self.keep_pages = torch.zeros(P, rows, dtype=torch.int32, device=device)
        self.pages = []
        for s, n in enumerate(need):
            own, order = order[:n], order[n:]
            self.pages.append(own)
            self.table[s, :n] = _ints(own, device)
            for i, p in enumerate(own):
                here = slice(i * rows, min((i + 1) * rows, lengths[s]))
                m = here.stop - here.start
                self.k_pages[p, :m], self.v_pages[p, :m] = self.k[s, here], self.v[s, here]
                if bias:
                    self.position_pages[p, :m] = self.key_positions[s, here]
                if keep:
                    self.keep_pages[p, :m] = self.keep[s, here]
        self.device_lengths = _ints(lengths, device)

    def run(self, **more):
        a = dict(q=self.q, k_pages=self.k_pages, v_pages=self.v_pages, page_table=self.table,
                 lengths=self.device_lengths, cap=self.cap, positions=self.positions,
                 position_pages=self.position_pages, slopes=self.slopes, keep_pages=self.keep_pages)
        return paged.paged_attention(**dict(a, **more))

    def scene(self, s, gone=()):
        """(value, bound) of scene s in 64 bits; rows of `gone` pages (by place) are not there."""
        n = self.lengths[s]
        live = [j for j in range(n) if j // self.rows not in gone]
        ref = dict(q_positions=self.positions[s:s + 1], k_positions=self.key_positions[s, live],
                   slopes=self.slopes) if self.slopes is not None else {}
        if self.keep is not None:
            ref["keep"] = self.keep[s, live]
        val, tol = R.attention(self.q[s:s + 1], self.k[s, live], self.v[s, live], cap=self.cap, **ref)
        return val["out"], tol["out"]

    def check(self, got, scenes=None, gone=()):
        assert got.shape == self.q.shape and got.dtype == self.q.dtype
        for s in range(len(self.lengths)) if scenes is None else scenes:
            val, tol = self.scene(s, gone)
            R.assert_within(got[s:s + 1], val, tol, f"scene {s} of {self.lengths[s]} rows")
        return got


# ---- attention


@TYPES
@pytest.mark.parametrize("dim", [8, 32, 40, 64, 96, 128])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (30.0, True)], ids=["plain", "cap, bias"])
@pytest.mark.parametrize("rows", [16, 48])
def test_lengths(device, route, dtype, dim, cap, bias, rows):
    """From none to a few hundred rows, ends inside a page and a step, beside each other."""
    c = Case(device, dtype, [0, 1, 2, 15, 16, 17, 31, 33, 64, 200, 0, 129], 4, 2, dim, rows=rows, cap=cap, bias=bias)
    got = c.check(c.run())
    assert not got[0].any() and not got[10].any()
    assert torch.equal(got[1], c.v[1, 0].repeat_interleave(2, 0))  # one row: its value
    assert torch.equal(got, c.run())


@TYPES
@pytest.mark.parametrize("lengths", [[5000], [1, 3000, 64], [700] * 9, [20_000] + [10] * 30],
                         ids=["one", "three", "even", "uneven"])
@pytest.mark.parametrize("heads", [(1, 1), (8, 2), (40, 1)], ids=["1", "8 on 2", "40 on 1"])
def test_rows_that_are_split(device, dtype, lengths, heads):
    c = Case(device, dtype, lengths, *heads, 64, rows=32)
    c.check(c.run(), scenes=range(min(len(lengths), 4)))


@TYPES
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("cap", [0.0, 30.0, 1e4])
@pytest.mark.parametrize("bias", [False, True])
def test_variants(device, dtype, dim, cap, bias):
    """Every kernel there is, over thousands of steps of a wave's pages."""
    c = Case(device, dtype, [16_500, 300], 2, 1, dim, cap=cap, bias=bias, rows=16)
    c.check(c.run())


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (50.0, True)])
def test_rounded_once(device, dim, cap, bias):
    """bfloat16 results are as exact as their type, over few rows and many."""
    c = Case(device, BF16, [2, 3, 9, 60, 127, 129, 1000, 9000], 32, 4, dim, cap=cap, bias=bias, rows=64)
    got = c.run()
    for s in range(len(c.lengths)):
        assert_rounded_once(got[s:s + 1], c.scene(s)[0], s)


@TYPES
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_as_over_rows_that_lie_together(device, dtype, dim):
    """The same rows over pages and together, both within their bounds."""
    c = Case(device, dtype, [200] * 4, 4, 2, dim, cap=20.0, rows=48)
    together = attention.cached_attention(c.q, c.k, c.v, c.device_lengths, cap=20.0, positions=c.positions,
                                          key_positions=c.key_positions, slopes=c.slopes)
    val = [c.scene(s) for s in range(4)]
    for got in (c.run(), together):
        for s, (v, t) in enumerate(val):
            R.assert_within(got[s:s + 1], v, t, s)


@TYPES
@pytest.mark.parametrize("scenes", [63, 64, 65, 130, 700])
def test_many_scenes(device, dtype, scenes):
    """More scenes than a wave has lanes, empty ones and long ones among them."""
    lengths = [(37 * s) % 90 * (s % 3 > 0) for s in range(scenes)]
    lengths[scenes // 2], lengths[-1] = 2500, 333
    c = Case(device, dtype, lengths, 2, 2, 32, bias=False)
    got = c.run()
    some = sorted({0, 1, 2, 3, scenes // 2, scenes - 2, scenes - 1} | set(range(5, scenes, 41)))
    c.check(got, scenes=some)
    empty = [s for s in range(scenes) if not lengths[s]]
    assert not got[empty].any() and torch.isfinite(got).all()


@TYPES
@pytest.mark.parametrize("heads,dim", [((16, 8), 128), ((8, 8), 64), ((6, 3), 40), ((17, 1), 32), ((64, 2), 96), ((32, 32), 8)],
                         ids=lambda x: str(x))
@pytest.mark.parametrize("lengths", [[900, 33, 0, 2000, 1, 150] * 9, [64] * 40 + [5000], [3000] * 4],
                         ids=["many", "long last", "few"])
def test_heads_and_cuts(device, dtype, heads, dim, lengths):
    """Few and many heads of one key head, that share lines of memory and that do not, in batches that are cut by
    scenes and by equal shares."""
    c = Case(device, dtype, lengths, *heads, dim, rows=64, cap=20.0)
    c.check(c.run(), scenes=[0, 1, 2, 3, len(lengths) - 1])
    alone = c.run(keep_pages=torch.ones(c.k_pages.shape[:2], dtype=torch.bool, device=device))
    assert torch.equal(alone, c.run())  # a mask that hides nothing, the same bits


@TYPES
def test_no_room_and_no_scenes(device, route, dtype):
    c = Case(device, dtype, [40, 20], 4, 2, 64)
    assert not c.run(page_table=c.table[:, :0]).any()
    got = c.run(q=c.q[:0], page_table=c.table[:0], lengths=c.device_lengths[:0], positions=c.positions[:0])
    assert got.shape == (0, 4, 64)


@TYPES
def test_a_scene_does_not_depend_on_others_values(device, dtype):
    """Other scenes' values, of the same lengths, change no bit."""
    a, b = (Case(device, dtype, [900, 20, 0, 333], 4, 2, 64, seed=s) for s in (1, 2))
    for n in ("q", "positions"):
        getattr(b, n)[3] = getattr(a, n)[3]
    for i, p in enumerate(b.pages[3]):
        for n in ("k_pages", "v_pages", "position_pages"):
            getattr(b, n)[p] = getattr(a, n)[a.pages[3][i]]
    assert torch.equal(a.run()[3], b.run()[3])


@TYPES
@pytest.mark.parametrize("bad", [-1, -(2**31), 2**31 - 1, "pages"])
@pytest.mark.parametrize("rows", [16, 32])
def test_entries_that_name_no_page(device, route, dtype, bad, rows):
    """Their rows are not there, in the middle of a scene, at its start, or all of them."""
    for gone in ([2], [0], [0, 1, 5], list(range(20))):
        c = Case(device, dtype, [300, 77], 4, 2, 64, rows=rows, cap=20.0)
        for i in gone:
            if i < c.table.shape[1]:
                c.table[:, i] = c.k_pages.shape[0] if bad == "pages" else bad
        got = c.check(c.run(), gone=gone)
        if len(gone) == 20:
            assert not got.any()


@TYPES
@pytest.mark.parametrize("keep_type", [torch.int32, torch.bool, torch.uint8])
@pytest.mark.parametrize("share", [0.3, 1.1], ids=["some", "all"])
def test_masked_keys(device, route, dtype, keep_type, share):
    """What masked rows hold (infinities, NaN, the lowest value) reaches nothing; a scene with all keys masked gives 0."""
    c = Case(device, dtype, [0, 1, 40, 333, 2000], 4, 2, 64, keep=share, rows=48)
    for s, own in enumerate(c.pages):
        for i, p in enumerate(own):
            for r in range(min(c.rows, c.lengths[s] - i * c.rows)):
                if r % 7 < 3 and not c.keep_pages[p, r]:
                    x = (float("nan"), float("inf"), torch.finfo(dtype).min)[r % 7]
                    c.k_pages[p, r], c.v_pages[p, r] = x, x
    got = c.check(c.run(keep_pages=(c.keep_pages != 0).to(keep_type)))
    if share > 1:
        assert not got.any()


@TYPES
@pytest.mark.parametrize("joint", [False, True])
def test_pools_as_they_lie(device, route, dtype, joint):
    """Halves of one pool, heads before rows, wide rows, a table and positions out of wider arrays."""
    c = Case(device, dtype, [100, 260, 5], 4, 2, 40, rows=32, joint=joint, room=3)
    want = c.run()
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.k_pages, c.v_pages)]
    wide = [torch.cat((t, t), -1)[..., :40] for t in (c.k_pages, c.v_pages)]
    places = torch.cat((c.position_pages, c.position_pages), -1)[..., :3]
    table = torch.cat((c.table, c.table), 1)[:, :c.table.shape[1]]
    for k, v in (heads_first, wide):
        assert torch.equal(c.run(k_pages=k, v_pages=v, position_pages=places, page_table=table), want)
    assert torch.equal(c.run(page_table=c.table.t().contiguous().t()), want)
    q = torch.cat((c.q, c.q), 2)[..., :40]
    assert torch.equal(c.run(q=q), want)
    assert torch.equal(c.run(q=c.q.transpose(1, 2).contiguous().transpose(1, 2)), want)


@TYPES
def test_shared_pages(device, dtype):
    """Scenes that begin alike hold those pages once."""
    c = Case(device, dtype, [160, 160, 160], 4, 2, 64)
    for s in (1, 2):
        c.table[s, :7] = c.table[0, :7]
        c.k[s, :112], c.v[s, :112], c.key_positions[s, :112] = c.k[0, :112], c.v[0, :112], c.key_positions[0, :112]
    c.check(c.run())


@TYPES
def test_lengths_past_the_table_and_below_zero(device, route, dtype):
    c = Case(device, dtype, [96, 96, 96], 4, 2, 64)
    got = c.run(lengths=_ints([2**31 - 1, -5, 97], device))
    c.check(got, scenes=[0, 2])
    assert not got[1].any()


@TYPES
def test_a_table_with_room(device, dtype):
    """Room for far more rows than there are costs no exactness."""
    c = Case(device, dtype, [500, 3, 40], 4, 2, 64, room=60_000, rows=16)
    c.check(c.run())


def test_pools_past_32_bits(device):
    """More than 2^32 elements: pages at both ends."""
    rows, K, D = 64, 8, 128
    P = 2**32 // (rows * K * D) + 50
    k, v = (torch.empty(P, rows, K, D, dtype=BF16, device=device) for _ in "kv")
    places = torch.empty(P, rows, 3, device=device)
    c = Case(device, BF16, [150, 128], 8, 8, D, rows=rows)
    ids = [P - 1, 3, P - 2, P // 2, P - 40]
    at = 0
    for s, own in enumerate(c.pages):
        for i, p in enumerate(own):
            k[ids[at]], v[ids[at]], places[ids[at]] = c.k_pages[p], c.v_pages[p], c.position_pages[p]
            c.table[s, i] = ids[at]
            at += 1
    c.check(c.run(k_pages=k, v_pages=v, position_pages=places))
    new = torch.randn(2, 8, D, generator=_gen(device, 3), device=device).to(BF16)
    far = torch.rand(2, 3, device=device)
    f = rotary.axis_frequencies((22, 21, 21), device=device)
    assert int(c.table[0, 2]) == P - 2
    paged.append_tokens(new, new, k, v, c.table, _ints([151, 1], device), positions=far, frequencies=f,
                        position_pages=places)
    turned = rotary.rotate_qk(new, new, far, f)[1]
    assert torch.equal(v[P - 2, 22], new[0]) and torch.equal(k[P - 2, 22], turned[0])
    assert torch.equal(places[P - 2, 22], far[0]) and torch.equal(v[int(c.table[1, 0]), 0], new[1])


@TYPES
def test_clear_winners_and_far_positions(device, dtype):
    c = Case(device, dtype, [700, 90], 4, 2, 64, spread=256.0, cap=50.0)
    c.q = c.q * 4
    got = c.check(c.run())
    for offset in (1e5, 1e6):
        c.positions, c.key_positions = c.positions + offset, c.key_positions + offset
        c.position_pages = c.position_pages + offset
        got = c.run()
        for s in range(2):
            val, tol = c.scene(s)
            R.assert_within(got[s:s + 1], val, tol, f"offset {offset}")
            if dtype == BF16:
                assert_rounded_twice(got[s:s + 1], val, s)


# ---- appending


class Tokens:
    """New tokens of some scenes, and the cache that takes them."""

    def __init__(self, device, dtype, counts, before, H, K, D, rows=16, axes=3, pairs=None, joint=False, seed=0,
                 single=False):
        g = _gen(device, seed)
        T, S = sum(counts), len(counts)
        self.counts, self.lengths, self.rows = counts, [n + b for n, b in zip(counts, before)], rows
        self.qkv = torch.randn(T, H + 2 * K, D, generator=g, device=device).to(dtype)
        self.q, self.k, self.v = self.qkv[:, :H], self.qkv[:, H:H + K], self.qkv[:, H + K:]
        self.positions = 256 * torch.rand(T, axes, generator=g, device=device)
        self.frequencies = torch.rand(axes, pairs or D // 2, generator=g, device=device)
        need = [-(-n // rows) for n in self.lengths]
        P = sum(need) + 3
        order = torch.randperm(P, generator=g, device=device).tolist()
        self.table = torch.full((S, max(max(need), 1)), -1, dtype=torch.int32, device=device)
        for s, n in enumerate(need):
            self.table[s, :n] = _ints(order[:n], device)
            order = order[n:]
        pool = torch.randn(P, 2, rows, K, D, generator=g, device=device).to(dtype)
        self.k_pages, self.v_pages = (pool[:, 0], pool[:, 1]) if joint else (pool[:, 0].clone(), pool[:, 1].clone())
        self.position_pages = torch.rand(P, rows, 3, generator=g, device=device)
        cuts = [0]
        for n in counts:
            cuts.append(cuts[-1] + n)
        self.starts = None if single else _ints(cuts, device)
        self.device_lengths = _ints(self.lengths, device)

    def targets(self):
        """(token, page, row in it) of the tokens that have a row."""
        t, table = 0, self.table.tolist()
        P, most = self.k_pages.shape[0], self.table.shape[1]
        for s, (n, length) in enumerate(zip(self.counts, self.device_lengths.tolist())):
            for i in range(n):
                j = length - n + i
                if 0 <= j < most * self.rows and 0 <= table[s][j // self.rows] < P:
                    yield t, table[s][j // self.rows], j % self.rows
                t += 1

    def want(self, interleaved=False, turn=True, places=True):
        k = self.k
        if turn:
            k = rotary.rotate_qk(self.k.contiguous(), self.k.contiguous(), self.positions, self.frequencies,
                                 interleaved=interleaved)[1]
        out = [self.k_pages.clone(), self.v_pages.clone(), self.position_pages.clone()]
        for t, p, r in self.targets():
            out[0][p, r], out[1][p, r] = k[t], self.v[t]
            if places:
                out[2][p, r] = self.positions[t]
        return out

    def run(self, **more):
        a = dict(k=self.k, v=self.v, k_pages=self.k_pages, v_pages=self.v_pages, page_table=self.table,
                 lengths=self.device_lengths, q=self.q, scene_starts=self.starts, positions=self.positions,
                 frequencies=self.frequencies, position_pages=self.position_pages)
        return paged.append_tokens(**dict(a, **more))

    def check(self, interleaved=False, **more):
        """The pools hold the tokens' rows, to the bit what rotary.rotate_qk gives, and are else as they were."""
        want = self.want(interleaved)
        q = self.run(interleaved=interleaved, **more)
        assert torch.equal(q, rotary.rotate_qk(self.q, None, self.positions, self.frequencies,
                                               interleaved=interleaved)[0])
        for got, w, what in zip((self.k_pages, self.v_pages, self.position_pages), want, "kvp"):
            assert torch.equal(got, w), what


@TYPES
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,pairs", [(8, 3), (16, 8), (40, 18), (40, 20), (64, 32), (64, 31), (96, 48), (128, 64),
                                       (128, 12)])
def test_append_sizes(device, route, dtype, interleaved, dim, pairs):
    Tokens(device, dtype, [3, 0, 17, 1, 40], [5, 9, 0, 15, 33], 5, 2, dim, pairs=pairs, rows=16).check(interleaved)


@TYPES
@pytest.mark.parametrize("dim", [40, 64])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_in_64_bits(device, dtype, dim, interleaved):
    """The turn against complex numbers in 64 bits.  The angle is rounded to binary32 within pi (2^-23 at most),
    sin and cos are 2^-23 off, products and sums three times 2^-24 of their size: in all 2^-21 of |x1| + |x2|."""
    c = Tokens(device, dtype, [33, 1], [0, 7], 3, 2, dim, rows=32)
    q = c.run(interleaved=interleaved)
    theta = c.positions.double() @ c.frequencies.double()
    w = torch.polar(torch.ones_like(theta), theta)[:, None]

    def turned(x):
        x = x.double()
        a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)
        z, size = torch.complex(a, b) * w, a.abs() + b.abs()
        if interleaved:
            return torch.view_as_real(z).flatten(-2), torch.stack((size, size), -1).flatten(-2)
        return torch.cat((z.real, z.imag), -1), torch.cat((size, size), -1)

    def near(got, x, what):
        val, size = turned(x)
        tol = 2.0 ** -21 * size + (0 if dtype == F32 else 2.0 ** -8) * (val.abs() + 2.0 ** -21 * size)
        R.assert_within(got, val, tol, what)

    near(q, c.q, "q")
    at = list(c.targets())
    near(torch.stack([c.k_pages[p, r] for _, p, r in at]), c.k[[t for t, _, _ in at]], "k")


@TYPES
@pytest.mark.parametrize("scenes", [1, 2, 16, 63, 300])
@pytest.mark.parametrize("rows", [16, 48, 256])
def test_append_one_token_a_scene(device, route, dtype, scenes, rows):
    before = [(29 * s) % 100 for s in range(scenes)]
    Tokens(device, dtype, [1] * scenes, before, 8, 2, 64, rows=rows, joint=True, single=True).check()


@TYPES
@pytest.mark.parametrize("counts", [[2000], [0] * 70 + [500] + [0] * 300 + [1, 2, 0, 700], [3] * 400,
                                    [1, 0] * 200 + [90], list(range(60))],
                         ids=["one", "far apart", "many", "in turn", "rising"])
@pytest.mark.parametrize("heads", [(2, 2), (12, 4)], ids=["2", "12 on 4"])
def test_append_prompts(device, dtype, counts, heads):
    Tokens(device, dtype, counts, [(7 * s) % 20 for s in range(len(counts))], *heads, 32, rows=32).check()


@TYPES
def test_append_rows_that_are_none(device, route, dtype):
    """Below row 0 (a scene of length 0 in a fixed batch), past the table, and in entries that name no page."""
    c = Tokens(device, dtype, [20, 20, 20, 1, 1], [0, 5, 40, 0, 3], 4, 2, 64)
    c.device_lengths = _ints([7, 0, 2**31 - 1, -4, 4], device)
    c.table[0, 0], c.table[4, 0] = c.k_pages.shape[0], -(2**31)
    c.check()
    assert not list(c.targets())
    c = Tokens(device, dtype, [40, 40], [0, 100], 4, 2, 64)
    c.device_lengths = _ints([25, 150], device)  # the first 15 tokens below row 0, the last 6 past the table
    c.table[0, 0] = -1
    c.check()
    assert 0 < len(list(c.targets())) < 80


@TYPES
@pytest.mark.parametrize("keep_type", [torch.int32, torch.bool, torch.uint8])
@pytest.mark.parametrize("pool_type", [torch.int32, torch.bool, torch.uint8])
def test_append_what_is_kept(device, route, dtype, keep_type, pool_type):
    c = Tokens(device, dtype, [9, 30], [1, 20], 4, 2, 64)
    keep = (torch.arange(39, device=device) % 3 * 5).to(keep_type)
    pool = (torch.arange(c.k_pages.shape[0] * 16, device=device).view(-1, 16) % 2).to(pool_type)
    want = pool.clone()
    for t, p, r in c.targets():
        want[p, r] = bool(keep[t])
    c.check(keep=keep, keep_pages=pool)
    assert torch.equal(pool, want)


@TYPES
@pytest.mark.parametrize("axes", [1, 2, 3, 8])
def test_append_parts(device, route, dtype, axes):
    """Without queries, without the turn, without positions; angles of other axes."""
    def new():
        return Tokens(device, dtype, [9, 30], [1, 20], 4, 2, 64, axes=axes)

    c = new()
    want = c.want(places=False)
    assert c.run(q=None, position_pages=None) is None
    assert torch.equal(c.k_pages, want[0]) and torch.equal(c.v_pages, want[1])
    c = new()
    want = c.want(turn=False, places=False)
    assert c.run(q=None, positions=None, frequencies=None, position_pages=None) is None
    assert torch.equal(c.k_pages, want[0]) and torch.equal(c.v_pages, want[1])
    if axes == 3:
        c = new()
        want = c.want(turn=False)
        assert c.run(q=None, frequencies=None) is None
        for got, w in zip((c.k_pages, c.v_pages, c.position_pages), want):
            assert torch.equal(got, w)


@TYPES
def test_append_views(device, route, dtype):
    """Copies where rows are off alignment or strided, pools with heads first, positions out of wider rows."""
    base = Tokens(device, dtype, [9, 30], [1, 20], 4, 2, 40)
    want, q = base.want(), None
    for n in range(4):
        c = Tokens(device, dtype, [9, 30], [1, 20], 4, 2, 40)
        if n == 1:
            c.k, c.v = (torch.cat((t, t[..., :1]), -1)[..., :40] for t in (c.k, c.v))
            c.q = c.q.transpose(1, 2).contiguous().transpose(1, 2)
        if n == 2:
            c.k_pages, c.v_pages = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.k_pages, c.v_pages))
            c.position_pages = torch.cat((c.position_pages, c.position_pages), -1)[..., :3]
        if n == 3:
            c.positions = torch.cat((c.positions, c.positions), -1)[:, :3]
            c.table = c.table.t().contiguous().t()
            c.frequencies = c.frequencies.t().contiguous().t()
        got = c.run()
        q = got if q is None else q
        assert torch.equal(got, q), n
        for a, b in zip((c.k_pages, c.v_pages, c.position_pages), want):
            assert torch.equal(a, b), n


def test_append_nothing(device, route):
    c = Tokens(device, BF16, [0, 0], [5, 9], 4, 2, 64)
    c.check()


# ---- both, as they are used


def _decode(c, steps, dtype, device, H, K, D, rows):
    """Scenes that grow by a token a step: the cache in pages against caches that lie together."""
    g = _gen(device, 9)
    S, f = 3, rotary.axis_frequencies((D // 6, D // 6, D // 2 - 2 * (D // 6)), device=device)
    P = S * (-(-steps // rows)) + 1
    pool = torch.full((P, 2, rows, K, D), float("nan"), dtype=dtype, device=device)
    places = torch.full((P, rows, 3), float("nan"), device=device)
    order = torch.randperm(P, generator=g, device=device)[:P - 1].int()
    table = torch.full((S, -(-steps // rows)), -1, dtype=torch.int32, device=device)
    k_all, v_all = (torch.zeros(S, steps, K, D, dtype=dtype, device=device) for _ in "kv")
    p_all, lengths = torch.zeros(S, steps, 3, device=device), torch.zeros(S, dtype=torch.int32, device=device)
    slopes = torch.rand(H, generator=g, device=device)
    for t in range(steps):
        qkv = torch.randn(S, H + 2 * K, D, generator=g, device=device).to(dtype)
        pos = 40 * torch.rand(S, 3, generator=g, device=device)
        if t % rows == 0:  # a page more for each
            table[:, t // rows] = order[S * (t // rows):S * (t // rows) + S]
        lengths += 1
        q = paged.append_tokens(qkv[:, H:H + K], qkv[:, H + K:], pool[:, 0], pool[:, 1], table, lengths, q=qkv[:, :H],
                                positions=pos, frequencies=f, position_pages=places)
        got = paged.paged_attention(q, pool[:, 0], pool[:, 1], table, lengths, positions=pos, position_pages=places,
                                    slopes=slopes, cap=20.0)
        q2, k_all[:, t] = rotary.rotate_qk(qkv[:, :H], qkv[:, H:H + K], pos, f)
        v_all[:, t], p_all[:, t] = qkv[:, H + K:], pos
        assert torch.equal(q, q2)
        if t % 11 == 0 or t + 1 == steps:
            for s in range(S):
                val, tol = R.attention(q2[s:s + 1], k_all[s, :t + 1], v_all[s, :t + 1], cap=20.0, slopes=slopes,
                                       q_positions=pos[s:s + 1], k_positions=p_all[s, :t + 1])
                R.assert_within(got[s:s + 1], val["out"], tol["out"], (t, s))


@TYPES
@pytest.mark.parametrize("rows", [16, 32])
def test_token_by_token(device, route, dtype, rows):
    _decode(None, 70, dtype, device, 4, 2, 48, rows)


@TYPES
def test_a_prompt_then_tokens(device, dtype):
    """Prompts through scene_attention and into the cache; the next token over the cache is the causal pass's."""
    g, counts, H, K, D = _gen(device, 4), [50, 1, 120], 4, 2, 64
    T = sum(counts)
    f = rotary.axis_frequencies((11, 11, 10), device=device)
    x = torch.randn(T, H + 2 * K, D, generator=g, device=device).to(dtype)
    pos = 40 * torch.rand(T, 3, generator=g, device=device)
    starts = _ints([0, 50, 51, 171], device)
    q, k = rotary.rotate_qk(x[:, :H], x[:, H:H + K], pos, f)
    whole = attention.scene_attention(q, k, x[:, H + K:], scene_starts=starts, causal=True)
    pools = [torch.zeros(14, 16, K, D, dtype=dtype, device=device) for _ in "kv"]
    table = torch.randperm(14, generator=g, device=device)[:14].int()
    table = torch.stack([torch.cat((table[:4], table[:4])), torch.cat((table[4:5], table[:7])), table[5:13]])
    # all but each scene's last token as a prompt, turned already
    last = [49, 50, 170]
    rest = [t for t in range(T) if t not in last]
    paged.append_tokens(k[rest], x[rest, H + K:], *pools, table, _ints([49, 0, 119], device),
                        scene_starts=_ints([0, 49, 49, 168], device))
    n = _ints(counts, device)
    q1 = paged.append_tokens(x[last, H:H + K], x[last, H + K:], *pools, table, n, q=x[last, :H], positions=pos[last],
                             frequencies=f)
    got = paged.paged_attention(q1, *pools, table, n)
    assert torch.equal(q1, q[last])
    for i, (t, s0) in enumerate(zip(last, (0, 50, 51))):
        val, tol = R.attention(q[t:t + 1], k[s0:t + 1], x[s0:t + 1, H + K:])
        R.assert_within(got[i:i + 1], val["out"], tol["out"], i)
        R.assert_within(whole[t:t + 1], val["out"], tol["out"], i)


@TYPES
def test_captured_steps(device, dtype):
    """A step in a graph: replays go by the lengths, the table and the tokens that they find."""
    g, S, H, K, D, rows = _gen(device, 5), 3, 4, 2, 64, 16
    f = rotary.axis_frequencies((11, 11, 10), device=device)
    pool = torch.zeros(40, 2, rows, K, D, dtype=dtype, device=device)
    places = torch.zeros(40, rows, 3, device=device)
    table = torch.full((S, 12), -1, dtype=torch.int32, device=device)
    lengths = torch.zeros(S, dtype=torch.int32, device=device)
    x = torch.randn(S, H + 2 * K, D, generator=g, device=device).to(dtype)
    pos, slopes = torch.rand(S, 3, generator=g, device=device), torch.rand(H, generator=g, device=device)

    def step(pool, places):
        q = paged.append_tokens(x[:, H:H + K], x[:, H + K:], pool[:, 0], pool[:, 1], table, lengths, q=x[:, :H],
                                positions=pos, frequencies=f, position_pages=places)
        return paged.paged_attention(q, pool[:, 0], pool[:, 1], table, lengths, positions=pos, position_pages=places,
                                     slopes=slopes)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pool, places)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(pool, places)
    other = [pool.clone(), places.clone()]
    for t in range(40):
        x.copy_(torch.randn(x.shape, generator=g, device=device))
        pos.copy_(40 * torch.rand(pos.shape, generator=g, device=device))
        lengths += _ints([1, t % 2, 1], device)
        if t % rows == 0:
            table[:, t // rows] = _ints([3 * (t // rows) + i for i in (2, 0, 1)], device)
        graph.replay()
        want = step(*other)
        assert torch.equal(out, want) and torch.equal(pool, other[0]) and torch.equal(places, other[1]), t
        torch.cuda.synchronize()
    # more rows than a step of the graph's capture had, split over pieces
    table.copy_(torch.arange(36, device=device).int().view(3, 12))
    lengths.copy_(_ints([190, 30, 0], device))
    pool.normal_(generator=g), places.uniform_(generator=g)
    other = [pool.clone(), places.clone()]
    for _ in range(3):
        graph.replay()
        assert torch.equal(out, step(*other)) and torch.equal(pool, other[0])


def test_on_another_stream_and_two_at_once(device):
    """Each call's workspace is its own: calls on two streams, started together."""
    a, b = (Case(device, BF16, [3000, 100], 8, 2, 64, seed=s) for s in (1, 2))
    want = a.run(), b.run()
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(10):
        for c, s, g in zip((a, b), streams, got):
            with torch.cuda.stream(s):
                g.append(c.run())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


def test_autograd_sees_the_writes(device, route):
    """A backward whose saved values the append has changed raises."""
    c = Tokens(device, F32, [2, 2], [0, 0], 4, 2, 64)
    w = torch.ones(64, device=device, requires_grad=True)
    loss = (c.k_pages * w).sum()
    c.run()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        d = Tokens(device, F32, [2, 2], [0, 0], 4, 2, 64)
        d.run()
    assert torch.equal(d.k_pages.clone(), c.k_pages)


# ---- refusals


def _refuses(call, text, error=ValueError, **more):
    with pytest.raises(error, match=text):
        call(**more)


def test_attention_refuses(device):
    c = Case(device, BF16, [40, 20], 4, 2, 64)

    def no(text, error=ValueError, **more):
        _refuses(c.run, text, error, **more)

    pool = torch.zeros(9, 16, 2, 64, dtype=BF16, device=device)
    no("2-D int32", page_table=c.table.long())
    no("2-D int32", page_table=c.table[0])
    no("page_table holds", page_table=c.table[:1])
    no("page_table must be on", page_table=c.table.cpu())
    no("one shape", k_pages=c.k_pages[1:])
    no("multiple of 16 rows", k_pages=pool[:, :8], v_pages=pool[:, :8])
    no("multiple of 16 rows", k_pages=pool[:0], v_pages=pool[:0])
    no("must have 4 axes", k_pages=c.k_pages[0])
    no("must be torch.bfloat16", k_pages=c.k_pages.float(), v_pages=c.v_pages.float())
    no("16-byte aligned", k_pages=torch.zeros(9, 16, 2, 68, dtype=BF16, device=device)[..., :64], v_pages=pool)
    no("channels must be", q=c.q[..., :60], k_pages=pool[..., :60], v_pages=pool[..., :60])
    no("channels", q=c.q[..., :32])
    no("not a multiple", q=c.q[:, :3], slopes=None, positions=None, position_pages=None)
    no("lengths", lengths=c.device_lengths.long())
    no("lengths must hold", lengths=c.device_lengths[:1])
    no("slopes need", positions=None)
    no("slopes need", position_pages=None)
    no("positions need slopes", slopes=None)
    no("position_pages must have shape", position_pages=c.position_pages[1:])
    no("together", position_pages=c.position_pages.transpose(1, 2).contiguous().transpose(1, 2))
    no("keep_pages must have shape", keep_pages=torch.ones(3, 16, dtype=torch.bool, device=device))
    no("keep_pages must be", keep_pages=torch.ones(c.k_pages.shape[:2], device=device))
    no("scale", scale=-1.0)
    no("scale", scale=0)
    no("cap", cap=-1.0)
    no("no gradient here", q=c.q.clone().requires_grad_())
    no("no gradient here", k_pages=c.k_pages.clone().requires_grad_())
    with torch.no_grad():
        c.run(q=c.q.clone().requires_grad_())


def test_append_refuses(device):
    c = Tokens(device, BF16, [4, 2], [0, 3], 4, 2, 64)
    before = [t.clone() for t in (c.k_pages, c.v_pages, c.position_pages)]

    def no(text, error=ValueError, **more):
        _refuses(c.run, text, error, **more)

    no("one shape", v=c.v[1:])
    no("must be torch.bfloat16", v=c.v.float())
    no("k must be a CUDA", k=c.k.cpu())
    no("heads of", k_pages=c.k_pages[:, :, :1], v_pages=c.v_pages[:, :, :1])
    no("share memory", v_pages=c.k_pages)
    pool = torch.zeros(c.k_pages.shape[0] + 1, 16, 2, 64, dtype=BF16, device=device)
    no("share memory", k_pages=pool[:-1], v_pages=pool[1:])
    no("share memory", k_pages=pool[1:], v_pages=pool[:-1])
    no("share memory", k_pages=pool[:-1], v_pages=pool.view(-1)[16:-2032].view(-1, 16, 2, 64))
    no("several elements", k_pages=c.k_pages[:1].expand(5, -1, -1, -1), v_pages=c.v_pages[:5], position_pages=None)
    no("several elements", position_pages=c.position_pages[:1].expand(c.position_pages.shape))
    no("need scene_starts", scene_starts=None)
    no("scene_starts must hold", scene_starts=c.starts[:2])
    no("lengths must hold", lengths=c.device_lengths[:1])
    no("need positions", positions=None, q=None)
    no("positions need", frequencies=None, position_pages=None, q=None)
    no("q needs frequencies", frequencies=None)
    no("rows, got", positions=c.positions[1:])
    no("3 axes", positions=c.positions[:, :2], frequencies=c.frequencies[:2])
    no("axes", frequencies=c.frequencies[:2])
    no("do not fit", frequencies=torch.zeros(3, 33, device=device))
    no("q must have k's", q=c.q[..., :32])
    no("each other", keep=torch.ones(6, dtype=torch.bool, device=device))
    no("no gradient here", k=c.k.clone().requires_grad_())
    no("no gradient here", positions=c.positions.clone().requires_grad_())
    no("no gradient here", position_pages=c.position_pages.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda k: paged.append_tokens(k, c.v, c.k_pages, c.v_pages, c.table, c.device_lengths,
                                                      scene_starts=c.starts) or k, (c.k,), check_trace=False)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda k: paged.append_tokens(k, c.v, c.k_pages, c.v_pages, c.table, c.device_lengths,
                                                      scene_starts=c.starts) or k)(c.k[None])
    for t, w in zip((c.k_pages, c.v_pages, c.position_pages), before):
        assert torch.equal(t, w)


@TYPES
def test_plain_calls_take_the_native_functions(device, monkeypatch, dtype):
    assert _native.available
    log = []
    for name in ("append_tokens", "paged_attention"):
        def record(*args, call=getattr(_native, name)):
            out = call(*args)
            log.append(bool(out))
            return out
        monkeypatch.setattr(_native, name, record)
    for joint in (False, True):
        c = Tokens(device, dtype, [4, 2], [0, 3], 4, 2, 40, joint=joint)
        keep = torch.ones(6, dtype=torch.bool, device=device)
        kept = torch.zeros(c.k_pages.shape[:2], dtype=torch.int32, device=device)
        c.run(), c.run(keep=keep, keep_pages=kept), c.run(q=None), c.run(interleaved=True)
        c.run(q=None, frequencies=None), c.run(q=None, frequencies=None, positions=None, position_pages=None)
        d = Tokens(device, dtype, [1] * 3, [5, 0, 20], 4, 2, 40, single=True)
        d.run()
        a = Case(device, dtype, [40, 20, 300], 4, 2, 40, joint=joint, keep=0.5)
        a.run(), a.run(keep_pages=None), a.run(slopes=None, positions=None, position_pages=None), a.run(cap=5.0, scale=0.2)
    assert len(log) == 22 and all(log)


def test_append_refuses_tokens_that_lie_in_the_pools(device, route):
    c = Tokens(device, BF16, [4, 2], [0, 3], 4, 2, 64)
    rows = c.k_pages.view(-1, 2, 64)
    keeps = torch.zeros(c.k_pages.shape[:2], dtype=torch.bool, device=device)
    before = [t.clone() for t in (c.k_pages, c.v_pages, c.position_pages, keeps)]
    for more in (dict(k=rows[:6]), dict(v=rows[-6:]), dict(q=rows[3:9]), dict(v=c.v_pages.view(-1, 2, 64)[:6]),
                 dict(positions=c.position_pages.view(-1, 3)[-6:]), dict(keep=keeps.view(-1)[4:10], keep_pages=keeps)):
        _refuses(c.run, "must not lie in", ValueError, **more)
    for t, w in zip((c.k_pages, c.v_pages, c.position_pages, keeps), before):
        assert torch.equal(t, w)
    # memory side by side is apart: the pools and the tokens of one allocation
    P, n = c.k_pages.shape[0], c.k_pages[0].numel()
    arena = torch.randn((2 * P + 1) * n, device=device).to(BF16)
    c.k_pages, c.v_pages = arena[:2 * P * n].view(2, P, 16, 2, 64)
    c.k = arena[2 * P * n:].view(-1, 2, 64)[:6]
    c.check()


def test_tokens_that_fill_a_batch_are_one_more_scene(device, route):
    """Packed prompts of a fixed size: what is behind the last prompt is a scene of length 0, and not written."""
    c = Tokens(device, F32, [5, 20, 7], [0, 3, 0], 4, 2, 40)
    c.device_lengths[2] = 0
    assert sum(1 for _ in c.targets()) == 25
    c.check()
