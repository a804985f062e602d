"""Bounds in the 2-norm on what bfloat16 attention may be off, and its roundings in the oracle's arithmetic.

An element's bound has to allow for the worst of all roundings at once; over many elements they add in
quadrature, and these bounds tell one rounding from two, and two from three.
"""
import math

import torch

import token_reference as R

BF16 = torch.bfloat16


def off(got, want):
    """How far off in the 2-norm, against the value's."""
    return float((got.double() - want).norm() / want.norm().clamp_min(1e-30))


def rounded_once(want):
    """As exact as its own type: what the rounding of the exact values to bfloat16 takes, and a tenth of it
    (other values round elsewhere); weights, ds and out enter the products with 16 bits, 2^-17 of
    each term, times what cancels in ds (2^4 here)."""
    return 1.1 * off(want.to(BF16), want) + 2.0 ** -13


def rounded_twice(want):
    """The rounding of the results and, in quadrature, as much from weights and ds of 8 bits; and a tenth."""
    return 1.1 * 2 ** 0.5 * off(want.to(BF16), want) + 2.0 ** -13


def assert_rounded_once(got, want, what):
    assert off(got, want) <= rounded_once(want), (what, off(got, want), off(want.to(BF16), want))


def assert_rounded_twice(got, want, what):
    assert off(got, want) <= rounded_twice(want), (what, off(got, want), off(want.to(BF16), want))


# The slopes' gradient in binary32 (before its own rounding): weights are off by some 2^-18 (64 products and the
# exponential's scaling, at scores of 50), and what they leave of it is a sum of terms of both signs, as
# large as sqrt(keys that count) times it.
SLOPES = 2.0 ** -13


def rounded_head(q, k, v, see, slope, far, dout, whole_out=True, rests=True):
    """One head of one scene with bfloat16's roundings (weights, ds and out of 8 bits, results rounded), sums
    exact: out, dq, dk, dv, dslope.  Without `whole_out` D comes from the rounded output; without `rests`
    the slope's gradient keeps the rows' rests."""
    q, k, v, dout = (t.double() for t in (q, k, v, dout))

    def b(t):
        return t.to(BF16).double()

    scale = 1 / math.sqrt(q.shape[1])
    t = (scale * (q @ k.T) - slope.double() * far).masked_fill(~see, -math.inf)
    e = (t - t.amax(1, keepdim=True)).exp()
    p, w = e / e.sum(1, keepdim=True), b(e)
    o = w @ v / w.sum(1, keepdim=True)
    delta = (dout * (b(o) + (b(o - b(o)) if whole_out else 0))).sum(1, keepdim=True)
    dt = p * (dout @ v.T - delta)
    dslope = -(dt * far).sum()
    if rests:
        dslope = dslope + (dt.sum(1) * (p * far).sum(1)).sum()
    return dict(out=b(o), dq=b(scale * b(dt) @ k), dk=b(scale * b(dt).T @ q), dv=b(b(p).T @ dout),
                dslopes=dslope[None])


def clear_winners(tokens, dim, seed, causal):
    """One head of a scene whose rows have most of their weight on a few keys: rounded_head's arguments and
    the exact values."""
    g = torch.Generator().manual_seed(seed)
    q, k, v, dout = ((torch.randn(tokens, dim, generator=g) * (4 if n == 0 else 1)).to(BF16) for n in range(4))
    pos, slope = 256 * torch.rand(tokens, 3, generator=g), torch.tensor([1 / 32])
    see = R.seen(tokens, tokens, causal, 0, None, "cpu")
    far = (pos.double()[:, None] - pos.double()[None]).norm(dim=-1)
    val, _ = R.one_head(q, k, v, see, 1 / math.sqrt(dim), 0.0, slope[0], pos, pos, dout, BF16)
    val["dslopes"] = val.pop("dslope")[None]
    return (q, k, v, see, slope, far, dout), val
