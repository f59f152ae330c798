"""A gated feed-forward block and its gradients in 64 bits, with bounds on what 16-bit operands may be off by.

The bounds follow the kernels' roundings element by element.  u = finfo(dtype).eps / 2 is half a step, what one rounding may move a value by
relative to itself; a value under the smallest normal number moves by half of the smallest subnormal, `tiny`.  Sums of n products of
16-bit numbers are exact products added in 32 bits in any order: off by at most n 2^-24 (1 + small) of the sum of magnitudes; 2^-23 is
taken.  The gate is computed in 32 bits from a hardware exponential, reciprocal and a polynomial: `ARITH` of itself (2^-18) and 2^-21 absolute,
since g / ln 2 loses |g| 2^-24 in the exponent, GELU's Phi is 1.3e-7 off and for |g| < 16 that is more than all the roundings.  The bounds of
differences: |act'| <= 1.13, |act''| <= 0.8 for SiLU and GELU; ReLU's slope may be the other one where |g| is within its error.
"""
import math

import torch

ARITH, ABS = 2.0 ** -18, 2.0 ** -21
SLOPE, CURVE = 1.13, 0.8


def act(g, name):
    """The activation and its derivative."""
    if name == "relu":
        return g.clamp_min(0.0), (g > 0).double()
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1.0 - s)
    below = 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
    return g * below, below + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)


def keep(mask, bs, rows, cols, p, like):
    if mask is None:
        return torch.ones(rows, cols, dtype=torch.float64, device=like.device)
    wide = (~mask).double().repeat_interleave(bs, 0).repeat_interleave(bs, 1)[:rows, :cols]
    return wide / (1.0 - p)


def block(x, w_in, w_out, name, by_x, by_h):
    """y, in torch's autograd where it is asked for."""
    f = w_out.shape[1]
    a = (x * by_x) @ w_in.t()
    return (act(a[:, :f], name)[0] * a[:, f:] * by_h) @ w_out.t()


def reference(x, w_in, w_out, dy, name, dtype, masks=(None, None), bs=64, ps=(0.0, 0.0)):
    """{name: (value, bound)} of y, dx, dw_in, dw_out; operands are tensors in 16 bits."""
    u, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    # the scale of a product that drops is a float, 2^-24 of itself off, and multiplies once more
    fl = 2.0 ** -22
    x, w_in, w_out, dy = (t.detach().double() for t in (x, w_in, w_out, dy))
    (m, k), (n, f) = x.shape, w_out.shape
    by_x, by_h = keep(masks[0], bs, m, k, ps[0], x), keep(masks[1], bs, m, f, ps[1], x)

    def rounded(v, e):
        """e and one rounding of a value that is off by e."""
        return e + u * (v.abs() + e) + tiny

    def product(a, ea, b, eb):
        v = a @ b
        mag = a.abs() @ b.abs()
        return v, ea @ b.abs() + (a.abs() + ea) @ eb + (a.shape[1] * 2.0 ** -23 + fl) * (mag + ea @ (b.abs() + eb))

    def none(t):
        return torch.zeros_like(t)

    xd = x * by_x
    a, ea = product(xd, none(xd), w_in.t(), none(w_in.t()))
    ea = rounded(a, ea)
    g, up, eg, eu = a[:, :f], a[:, f:], ea[:, :f], ea[:, f:]
    v, s = act(g, name)
    ev = SLOPE * eg + ARITH * v.abs() + ABS
    es = CURVE * eg + ARITH * s.abs() + ABS
    if name == "relu":
        ev, es = eg, (g.abs() <= eg).double()
    h = v * up
    eh = rounded(h, ev * (up.abs() + eu) + v.abs() * eu + 2.0 ** -23 * h.abs())
    hd, ehd = h * by_h, eh * by_h
    y, ey = product(hd, ehd, w_out.t(), none(w_out.t()))
    dh, edh = product(dy, none(dy), w_out, none(w_out))
    dh, edh = dh * by_h, rounded(dh * by_h, edh * by_h) * (by_h > 0)
    dg = dh * up * s
    edg = (dh.abs() + edh) * (up.abs() + eu) * (s.abs() + es) * (1 + 2.0 ** -21) - dg.abs()
    du = dh * v
    edu = (dh.abs() + edh) * (v.abs() + ev) * (1 + 2.0 ** -22) - du.abs()
    da, eda = torch.cat((dg, du), 1), torch.cat((rounded(dg, edg), rounded(du, edu)), 1) * torch.cat((by_h > 0, by_h > 0), 1)
    dx, edx = product(da, eda, w_in, none(w_in))
    dw_in, edw_in = product(da.t(), eda.t(), xd, none(xd))
    dw_out, edw_out = product(dy.t(), none(dy.t()), hd, ehd)
    return {"y": (y, rounded(y, ey)), "dx": (dx * by_x, rounded(dx * by_x, edx * by_x) * (by_x > 0)), "dw_in": (dw_in, rounded(dw_in, edw_in)),
            "dw_out": (dw_out, rounded(dw_out, edw_out))}
