"""The token operators from their definitions, in 64 bits, with the error bounds that their kernels are held to (test infrastructure only).

Every function returns (value, bound) pairs: `bound` is what float32 arithmetic, and for bf16 tensors the roundings to bf16 that the kernels make, can move each value by."""
import math

import torch

U32, U16 = 2.0 ** -24, 2.0 ** -8          # half a unit in the last place, relative: float32, bf16


def _unit(dtype):
    return U16 if dtype == torch.bfloat16 else U32


def layer_norm(x, weight, bias, eps, dy=None, y_dtype=None):
    """y and, with dy, (y, dx, dweight, dbias) of layer norm over the last axis of x [rows, C], each with its bound."""
    xd, C, rows = x.double(), x.shape[-1], x.shape[0]
    w = torch.ones(C, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    mean = xd.mean(1, keepdim=True)
    var = (xd - mean).square().mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = (xd - mean) * r
    # a float32 sum of C terms is off by at most C * U32 of the terms' size; the mean's error shifts the row, the variance's scales it
    e_mean = (C + 4) * U32 * xd.abs().mean(1, keepdim=True)
    e_xh = r * (e_mean + 2 * U32 * (xd.abs() + mean.abs())) + xh.abs() * ((2 * C + 16) * U32 + r * r * e_mean * e_mean)
    y = xh * w + b
    uy = _unit(x.dtype if y_dtype is None else y_dtype)
    out = [(y, e_xh * w.abs() + 3 * U32 * (y.abs() + b.abs()) + uy * y.abs())]
    if dy is None:
        return out[0]
    g = dy.double() * w
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = r * (g - m1 - xh * m2)
    a1, a2 = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
    e = r * ((C + 16) * U32 * (a1 + xh.abs() * a2 + g.abs()) + e_xh * m2.abs() + xh.abs() * (g.abs() * e_xh).mean(1, keepdim=True))
    out.append((dx, e + dx.abs() * ((2 * C + 16) * U32 + _unit(x.dtype))))
    d = dy.double()
    out.append(((d * xh).sum(0), (d.abs() * e_xh).sum(0) + (rows + 8) * U32 * (d * xh).abs().sum(0)))
    out.append((d.sum(0), (rows + 8) * U32 * d.abs().sum(0)))
    return out


def rotary(x, positions, frequencies, pairs_per_axis, prefix=0, interleaved=False, inverse=False):
    P = sum(pairs_per_axis)
    axis = [a for a, n in enumerate(pairs_per_axis) for _ in range(n)]
    t = (positions.double()[..., axis] * frequencies.double()).unsqueeze(-2)
    if t.dim() == 3:
        t = t.unsqueeze(0)
    c, s = torch.cos(t), torch.sin(-t if inverse else t)
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    first = torch.arange(P, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else P)
    u, v = y[:, prefix:, :, first], y[:, prefix:, :, second]
    y[:, prefix:, :, first], y[:, prefix:, :, second] = u * c - v * s, v * c + u * s
    size[:, prefix:, :, first] = size[:, prefix:, :, second] = u.abs() + v.abs()
    # cos and sin to a few units in the last place, t^2 * U32^2 for the part of the angle that is turned to first order, two products and a sum
    e = size * (8 * U32 + (t.abs().max() * U32 if t.numel() else 0.0) ** 2)
    return y, e + (_unit(x.dtype) * y.abs() * (size > 0))


def attention(q, k, v, key_lengths=None, key_mask=None, scale=None, dy=None):
    """o and, with dy, (o, dq, dk, dv), each with its bound."""
    dt, (B, Lq, H, D), (Lk, G) = q.dtype, q.shape, k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    ok = torch.ones((B, Lk), dtype=torch.bool, device=q.device)
    if key_lengths is not None:
        ok &= torch.arange(Lk, device=q.device) < key_lengths[:, None]
    if key_mask is not None:
        ok &= key_mask
    def heads(t): return t.double().permute(0, 2, 1, 3)
    clean = ok[:, None, :, None]
    qd = heads(q)
    kd, vd = (torch.where(clean, heads(t), 0.0).repeat_interleave(H // G, 1) for t in (k, v))
    s = (qd @ kd.transpose(2, 3)) * scale
    s = s.masked_fill(~ok[:, None, None, :], float("-inf"))
    top = s.amax(-1, keepdim=True) if Lk else s.new_zeros(B, H, Lq, 1)
    e = torch.exp(s - torch.where(torch.isinf(top) & (top < 0), 0.0, top))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    o = p @ vd
    bf = dt == torch.bfloat16
    # float32: a score is off by (D + 4) U32 of its terms' size, its exponential by that much relatively, and so is the sum
    terms = (qd.abs() @ kd.abs().transpose(2, 3)).amax((-1, -2), keepdim=True) * abs(scale) if Lk else 0.0
    rel = 4 * (D + 8) * U32 * (terms + 1) + (Lk + 16) * U32
    step = U16 if bf else 0.0                     # the weights are rounded in front of the product with v
    size = p @ vd.abs()
    e_o = (rel + step) * size
    def back(t): return t.permute(0, 2, 1, 3)
    out = [(back(o), back(e_o + _unit(dt) * (o.abs() + e_o)))]
    if dy is None:
        return out[0]
    g = heads(dy)
    dp = g @ vd.transpose(2, 3)
    delta = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dpa = g.abs() @ vd.abs().transpose(2, 3)
    e_delta = (g.abs() * (e_o + _unit(dt) * (o.abs() + e_o))).sum(-1, keepdim=True) + (D + 4) * U32 * (g * o).abs().sum(-1, keepdim=True)
    e_ds = ds.abs() * (rel + step) + p * (e_delta + (D + 8) * U32 * (dpa + delta.abs()) * (1 + rel))
    n = (Lk + Lq * (H // G) + 16) * U32
    def state(t): return back(t.reshape(B, G, H // G, Lk, D).sum(2))
    dsa, pa = ds.abs() + e_ds, p
    grads = [(ds @ kd * scale, (e_ds @ kd.abs() + n * (dsa @ kd.abs())) * abs(scale), back),
             (ds.transpose(2, 3) @ qd * scale, (e_ds.transpose(2, 3) @ qd.abs() + n * (dsa.transpose(2, 3) @ qd.abs())) * abs(scale), state),
             (p.transpose(2, 3) @ g, (rel + step + n) * (pa.transpose(2, 3) @ g.abs()), state)]
    for value, err, form in grads:
        value, err = form(value), form(err)
        out.append((value, err + _unit(dt) * (value.abs() + err)))
    return out


def near(got, want):
    """Asserts that `got` lies within the bound of `want` = (value, bound), and that nothing in it is not a number."""
    value, bound = want
    assert got.shape == value.shape, (got.shape, value.shape)
    if not got.numel():
        return
    assert torch.isfinite(got).all()
    over = (got.double() - value).abs() - bound - 1e-37
    worst = int(over.reshape(-1).argmax())
    assert over.max() <= 0, f"value {got.reshape(-1)[worst].item()} at {worst}, wanted {value.reshape(-1)[worst].item()} +- {bound.reshape(-1)[worst].item()}"
