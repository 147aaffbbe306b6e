"""The operators of a token block (root-mean-square norm, 8-bit rows and their product, gated feed-forward) from their definitions, in 64 bits, with the error bounds that their
kernels are held to (test infrastructure only).

Functions return (value, bound) pairs, as in token_oracle: `bound` is what float32 arithmetic, and for bf16 tensors the roundings that the kernels make, can move each value by.
A float32 sum of n products is off by at most 2 (n + 8) U32 of the products' size: one rounding a step, of a whole unit where the adders of a matrix unit cut off."""
import math

import torch

from oracle.token_oracle import U16, U32, _unit, near  # noqa: F401

U24 = 2.0 ** -16              # the upper 24 bits of a float32, relative
TINY = torch.finfo(torch.float32).tiny


def rms_norm(x, weight, eps, residual=None, dy=None, dt=None):
    """[y, (total,) dx, dweight] (the gradients with dy; dt: the gradient of total), each with its bound."""
    total = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    t, C, rows, unit = total.double(), x.shape[-1], x.shape[0], _unit(x.dtype)
    w = torch.ones(C, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    r = 1 / torch.sqrt(t.square().mean(1, keepdim=True) + eps)
    th = t * r
    y = th * w
    rel = (C + 20) * U32                          # the sum of squares, its root, two products
    out = [(y, y.abs() * (rel + unit))]
    if residual is not None:
        out.append((t, torch.zeros_like(t)))
    if dy is None:
        return out
    d = dy.double()
    g = d * w
    m, size = (g * th).mean(1, keepdim=True), (g * th).abs().mean(1, keepdim=True)
    dx = r * (g - th * m)
    e = r * (g.abs() + th.abs() * size) * (2 * C + 48) * U32
    if dt is not None:
        dx = dx + dt.double()
        e = e + 4 * U32 * dt.double().abs()
    out.append((dx, e + unit * (dx.abs() + e)))
    out.append(((d * th).sum(0), (rows + C + 28) * U32 * (d * th).abs().sum(0)))
    return out


def eight_bits(y, e):
    """A row's scale with its bound, from values y that are off by at most e."""
    most = y.abs().amax(-1)
    scale = (most / 127).clamp_min(TINY)
    return scale, e.amax(-1) / 127 + 2 * U32 * scale


def near_eight_bits(q, scale, y, e):
    """Asserts that q * scale is y, off by at most e, to half a step of the given scale."""
    want, bound = eight_bits(y, e)
    near(scale, (want, bound))
    assert q.dtype is torch.int8 and q.shape == y.shape and (q >= -127).all()
    s = scale.double()[..., None]
    near(q.double() * s, (y, s * (0.5 + 130 * 4 * U32) + e))


def linear_int8(q, scale, weight, weight_scale, bias, out_dtype):
    y = (q.double() @ weight.double().T) * scale.double()[:, None] * weight_scale.double()
    b = torch.zeros_like(weight_scale, dtype=torch.float64) if bias is None else bias.double()
    e = 6 * U32 * (y.abs() + b.abs())
    y = y + b
    return y, e + _unit(out_dtype) * (y.abs() + e)


def feed_forward(x, gate_weight, up_weight, down_weight, gate_bias, up_bias, down_bias, activation, dy=None):
    """[y] or, with dy, [y, dx, dgate_weight, dup_weight, ddown_weight, dgate_bias, dup_bias, ddown_bias], each with its bound."""
    unit, bf = _unit(x.dtype), x.dtype == torch.bfloat16
    (F, C), O, M = gate_weight.shape, down_weight.shape[0], x.shape[0]
    step = U16 if bf else 0.0

    def of(n): return 2 * (n + 8) * U32
    def zero(b, n): return torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b.double()
    xd, wg, wu, wd = (t.double() for t in (x, gate_weight, up_weight, down_weight))
    bg, bu, bd = zero(gate_bias, F), zero(up_bias, F), zero(down_bias, O)
    g, u = xd @ wg.T + bg, xd @ wu.T + bu
    eg, eu = of(C) * (xd.abs() @ wg.abs().T + bg.abs()), of(C) * (xd.abs() @ wu.abs().T + bu.abs())
    if activation == "silu":
        p = torch.sigmoid(g)
        slope = p * (1 + g * (1 - p))
    else:
        p = 0.5 * torch.erfc(-g / math.sqrt(2))
        slope = p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    a = g * p
    # the functions themselves: an exponential whose argument is rounded, a quotient; an error function to an absolute unit; both curve by less than 1
    e_fn = (2 * g.abs() + 16) * U32 * a.abs() + 4 * U32 * g.abs()
    ea = slope.abs() * eg + eg * eg + e_fn
    h = a * u
    eh = ea * u.abs() + a.abs() * eu + ea * eu + 4 * U32 * h.abs()
    eh = eh + step * (h.abs() + eh)
    y = h @ wd.T + bd
    ey = eh @ wd.abs().T + of(F) * ((h.abs() + eh) @ wd.abs().T + bd.abs())
    out = [(y, ey + unit * (y.abs() + ey))]
    if dy is None:
        return out
    d = dy.double()
    if bf:                                        # g and u as the backward pass has them
        eg, eu = eg + U24 * (g.abs() + eg), eu + U24 * (u.abs() + eu)
    ea = slope.abs() * eg + eg * eg + e_fn
    es = 1.2 * eg + 8 * (g.abs() + 4) * U32
    dh = d @ wd
    edh = of(O) * (d.abs() @ wd.abs())

    def product(*pairs):
        """A product's value and bound from those of its factors, rounded as the hidden gradients are."""
        v, s = 1.0, 1.0
        for value, e in pairs:
            v, s = v * value, s * (value.abs() + e)
        e = s * (1 + 4 * U32) - v.abs()
        return v, e + step * (v.abs() + e)
    dg, edg = product((dh, edh), (u, eu), (slope, es))
    du, edu = product((dh, edh), (a, ea))
    dga, dua, ha = dg.abs() + edg, du.abs() + edu, h.abs() + eh
    results = [(dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs() + of(2 * F) * (dga @ wg.abs() + dua @ wu.abs())),
               (dg.T @ xd, edg.T @ xd.abs() + of(M) * (dga.T @ xd.abs())),
               (du.T @ xd, edu.T @ xd.abs() + of(M) * (dua.T @ xd.abs())),
               (d.T @ h, d.abs().T @ eh + of(M) * (d.abs().T @ ha)),
               (dg.sum(0), edg.sum(0) + of(M) * dga.sum(0)),
               (du.sum(0), edu.sum(0) + of(M) * dua.sum(0)),
               (d.sum(0), of(M) * d.abs().sum(0))]
    return out + [(v, e + unit * (v.abs() + e)) for v, e in results]
