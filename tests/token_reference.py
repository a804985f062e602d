"""The operators on packed tokens in binary64, from their definitions, and bounds on
what binary32 arithmetic and bfloat16 operands may be off from them.

bfloat16 keeps 8 significant bits: rounding a value moves it by at most 2^-8 of it
(float32: 2^-24).  The bounds add up the roundings that the operators document; they are
elementwise, and hold for any inputs.
"""
import math

import torch

ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def spans(starts, tokens):
    """Row ranges of the scenes."""
    if starts is None:
        return [(0, tokens)]
    cuts = [0] + [int(x) for x in starts[1:-1]] + [tokens]
    return list(zip(cuts, cuts[1:]))


def seen(nq, nk, causal, prefix, keep, device):
    """(nq, nk): the keys that each row of a scene sees."""
    see = torch.ones(nq, nk, dtype=torch.bool, device=device)
    if causal:
        i = torch.arange(nq, device=device)[:, None] + nk - nq
        j = torch.arange(nk, device=device)[None, :]
        see = (j <= i) | (j < prefix)
    if keep is not None:
        see = see & (keep != 0)[None, :]
    return see


def one_head(q, k, v, see, scale, cap, slope, qp, kp, dout=None, dtype=torch.float32):
    """One head of one scene in binary64: (values, bounds), dicts of out and, with dout, dq, dk,
    dv, dslope.  Keys that no row may see are replaced by zeros first: nothing of theirs counts."""
    q, k, v = q.double(), k.double(), v.double()
    any_row = see.any(0)
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    k, v = (torch.where(any_row[:, None], t, zero) for t in (k, v))
    raw = scale * (q @ k.T)
    size = scale * (q.abs() @ k.abs().T)
    t = cap * torch.tanh(raw / cap) if cap else raw
    far = torch.zeros_like(t)
    if slope is not None:
        kp = torch.where(any_row[:, None], kp.double(), zero)
        far = (qp.double()[:, None] - kp[None]).norm(dim=-1)
        t = t - slope.double() * far
    t = t.masked_fill(~see, -math.inf)
    top = t.amax(1, keepdim=True) if t.shape[1] else t.new_zeros(t.shape[0], 1)
    e = torch.exp(t - torch.where(top == -math.inf, zero, top))
    total = e.sum(1, keepdim=True)
    p = e / torch.where(total == 0, zero + 1, total)
    o = p @ v
    # a score's error: D products and sums in binary32, the bias, the exponent's scaling and
    # the exponential itself; a weight's relative error twice that (numerator, sum)
    u32, D, n = 2.0 ** -24, q.shape[1], max(k.shape[0], 1)
    u = ROUND[dtype]
    um = u if dtype != torch.float32 else 0.0  # operands of the matrix products
    tops = t.abs().masked_fill(~see, 0).amax() if t.numel() else zero
    biggest = size.masked_fill(~see, 0).amax() if t.numel() else zero
    s = slope.double().abs() if slope is not None else 0.0
    far_top = far.masked_fill(~see, 0).amax() if t.numel() else zero
    et = u32 * ((D + 4) * biggest + 8 * tops + 8 * s * far_top + 4 * cap + 8)
    ep = 2 * et + u32 * (n + 8)
    val, tol = {"out": o}, {"out": u * o.abs() + (um + ep) * 1.01 * (p @ v.abs()) + 1e-30}
    if dout is None:
        return val, tol
    g = dout.double()
    dp = g @ v.T
    delta = (g * o).sum(1, keepdim=True)
    dt = p * (dp - delta)
    curve = 1 - torch.tanh(raw / cap) ** 2 if cap else torch.ones_like(raw)
    ds = dt * curve
    val.update(dq=scale * ds @ k, dk=scale * ds.T @ q, dv=p.T @ g, dslope=-(dt * far).sum())
    # errors of dp (D products), of delta (from the rounded out), of p, and of ds's rounding
    e_dp = u32 * (D + 4) * (g.abs() @ v.abs().T)
    e_delta = ((tol["out"] * g.abs()).sum(1, keepdim=True)
               + u32 * (D + 4) * (g.abs() * o.abs()).sum(1, keepdim=True))
    e_dt = p * (e_dp + e_delta) + ep * dt.abs()
    e_curve = 4 * et / cap if cap else 0.0
    e_ds = e_dt * curve + dt.abs() * e_curve + (um + 4 * u32) * ds.abs()
    acc = u32 * (n + q.shape[0] + 8)
    tol["dq"] = scale * 1.01 * ((e_ds + acc * ds.abs()) @ k.abs()) + u * val["dq"].abs() + 1e-30
    tol["dk"] = scale * 1.01 * ((e_ds + acc * ds.abs()).T @ q.abs()) + u * val["dk"].abs() + 1e-30
    tol["dv"] = (um + ep + acc) * 1.01 * (p.T @ g.abs()) + u * val["dv"].abs() + 1e-30
    tol["dslope"] = 1.01 * ((e_dt + acc * dt.abs()) * far).sum() + u32 * 8 * (dt.abs() * far).sum()
    return val, tol


def attention(q, k, v, q_starts=None, k_starts=None, causal=False, prefix=None, scale=None, cap=0.0,
              slopes=None, q_positions=None, k_positions=None, keep=None, dout=None):
    """(values, bounds) of scene_attention's outputs: out, dq, dk, dv, dslopes."""
    T, H, D = q.shape
    N, K = k.shape[:2]
    scale = D ** -0.5 if scale is None else scale
    dev, f64 = q.device, torch.float64
    shapes = {"out": q.shape, "dq": q.shape, "dk": k.shape, "dv": v.shape, "dslopes": (H,)}
    names = ["out"] + (["dq", "dk", "dv", "dslopes"] if dout is not None else [])
    val, tol = ({n: torch.zeros(shapes[n], dtype=f64, device=dev) for n in names} for _ in "ab")
    ks = q_starts if k_starts is None else k_starts
    for s, ((q0, q1), (k0, k1)) in enumerate(zip(spans(q_starts, T), spans(ks, N))):
        see = seen(q1 - q0, k1 - k0, causal, 0 if prefix is None else int(prefix[s]),
                   None if keep is None else keep[k0:k1], dev)
        for h in range(H):
            hk = h // (H // K)
            a, b = one_head(q[q0:q1, h], k[k0:k1, hk], v[k0:k1, hk], see, scale, cap,
                            None if slopes is None else slopes[h],
                            None if slopes is None else q_positions[q0:q1],
                            None if slopes is None else k_positions[k0:k1],
                            None if dout is None else dout[q0:q1, h], q.dtype)
            for x, y in ((val, a), (tol, b)):
                x["out"][q0:q1, h] = y["out"]
                if dout is not None:
                    x["dq"][q0:q1, h] = y["dq"]
                    x["dk"][k0:k1, hk] += y["dk"]
                    x["dv"][k0:k1, hk] += y["dv"]
                    x["dslopes"][h] += y["dslope"]
    if dout is not None and slopes is not None:
        tol["dslopes"] += ROUND[slopes.dtype] * val["dslopes"].abs()
    return val, tol


def assert_within(got, val, tol, what):
    """Every element of `got` is finite and within its bound of `val`."""
    assert tuple(got.shape) == tuple(val.shape), what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    if not got.numel():
        return
    over = (got.double() - val).abs() / tol.clamp_min(1e-300)
    i = int(over.argmax())
    assert float(over.max()) <= 1, (f"{what}: element {i} is {float(over.max()):.3g} bounds off: "
                                    f"{float(got.flatten()[i])} for {float(val.flatten()[i])}")
