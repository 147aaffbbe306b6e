"""Operators on tokens, for what stands behind a foveated patch embedding: layer norm, rotary positions with several axes, cross attention to an encoder's
states of another length, root-mean-square norm with the residual's addition, and the gated feed-forward block, each with its gradients; and for serving tokens and weights in 8 bits
and their product.  All on the library's own kernels.

In the reference they are torch calls inside its vision transformers (fovi/arch/vit.py:351-381: attention; fovi/arch/knnvit.py:420-464: rotary positions from the
tokens' sensor coordinates).  Here

* ``layer_norm`` / ``rotary`` / ``cross_attention`` / ``rms_norm`` / ``gated_feed_forward`` are differentiable functions of tensors,
* ``TokenNorm`` / ``AxialRotary`` / ``CrossAttention`` / ``TokenRMSNorm`` / ``GatedFeedForward`` the modules around them,
* ``rms_norm_int8`` / ``quantize`` / ``linear_int8`` serve in 8 bits, without gradients, and ``Linear8`` is a linear layer in that form, and
* ``FixationReader`` runs them together: the tokens of all fixations of an image become states with a place (time, height, width) of their own, and a set of learned queries
  reads them out.

CUDA tensors, float32 or bf16; there is no CPU path.
"""
import math

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops

__all__ = ["layer_norm", "rotary", "cross_attention", "rms_norm", "rms_norm_int8", "quantize", "linear_int8", "gated_feed_forward", "TokenNorm", "AxialRotary", "CrossAttention",
           "TokenRMSNorm", "GatedFeedForward", "Linear8", "FixationReader", "check"]


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _no_tangents(name, *tensors):
    """Forward-mode derivatives are not built: a tensor that carries one is refused, where the kernels would give a result without it, whose derivative reads as zero."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name}: forward-mode derivatives are not built; use backward-mode ones, or pass tensors without a tangent")


# ------------------------------------------------------------------------------------------------------------ functions
class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        y, stats = ops.layer_norm(x, weight, bias, eps, out_dtype, want_stats=True)
        ctx.save_for_backward(x, weight, stats)
        ctx.like = tuple(None if t is None else (t.dtype, t.shape) for t in (weight, bias))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, stats = ctx.saved_tensors
        dx, dw, db = ops.layer_norm_backward(x, grad, weight, stats, ctx.needs_input_grad[:3])
        dw, db = (None if g is None else g.to(like[0]).view(like[1]) for g, like in zip((dw, db), ctx.like))
        return dx, dw, db, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, out_dtype=None):
    """Layer norm over the last axis: y = (x - mean) / sqrt(var + eps) * weight + bias with the biased variance.  x [..., C] float32 or bf16; weight, bias [C] or
    None; the result has x's type, or `out_dtype`.  Statistics, sums and the parameters' gradients are float32; those gradients are the same bits every time."""
    if ops._native is not None and out_dtype is None and x.is_cuda:
        dev = ops._current_device()
        got = ops._native.layer_norm(x, weight, bias, eps, dev, ops._raw_stream(dev))
        if got is not None:
            return ops._checked(got, "fovi_layer_norm_forward")
    _no_tangents("layer_norm", x, weight, bias)
    if _wants_grad(x, weight, bias):
        return _LayerNormFunction.apply(x, weight, bias, eps, out_dtype)
    return ops.layer_norm(x, weight, bias, eps, out_dtype)


class _RotaryFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, frequencies, pairs_per_axis, prefix, interleaved):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = (pairs_per_axis, prefix, interleaved)
        return ops.rotary(x, positions, frequencies, pairs_per_axis, prefix, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return ops.rotary(grad, *ctx.saved_tensors, *ctx.how, inverse=True), None, None, None, None, None


_PAIRINGS = {"halves": False, "pairs": True}


def rotary(x, positions, frequencies, pairs_per_axis, prefix=0, pairing="halves"):
    """Rotary positions with several axes: pair p of every head of x [B, L, H, D] turns by position[axis of p] * frequencies[p].

    positions: float32 [L - prefix, axes] or [B, L - prefix, axes]; the first `prefix` tokens (class, registers) have no place and pass.  pairs_per_axis: how many of the
    pairs, in order, belong to each axis (1 to 4 axes).  frequencies: float32, one for each pair.  pairing: a pair is the channels (p, p + P) of the first 2P ("halves") or (2p, 2p + 1)
    ("pairs"); channels from 2P on pass.  Differentiable with respect to x; positions and frequencies carry no gradient."""
    if pairing not in _PAIRINGS:
        raise ValueError(f"pairing is {pairing!r}: 'halves' or 'pairs'")
    if ops._native is not None and x.is_cuda:
        dev = ops._current_device()
        got = ops._native.rotary(x, positions, frequencies, pairs_per_axis, prefix, _PAIRINGS[pairing], dev, ops._raw_stream(dev))
        if got is not None:
            return ops._checked(got, "fovi_rotary")
    _no_tangents("rotary", x, positions, frequencies)
    if _wants_grad(positions, frequencies):
        raise NotImplementedError("rotary: positions and frequencies carry no gradient; detach them")
    if _wants_grad(x):
        return _RotaryFunction.apply(x, positions, frequencies, pairs_per_axis, prefix, _PAIRINGS[pairing])
    return ops.rotary(x, positions, frequencies, pairs_per_axis, prefix, _PAIRINGS[pairing])


class _AttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_lengths, key_mask, scale):
        o, lse = ops.attention(q, k, v, key_lengths, key_mask, scale, want_lse=True)
        ctx.save_for_backward(q, k, v, o, lse, key_lengths, key_mask)
        ctx.scale = scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, o, lse, key_lengths, key_mask = ctx.saved_tensors
        return ops.attention_backward(q, k, v, o, grad, lse, key_lengths, key_mask, ctx.scale, ctx.needs_input_grad[:3]) + (None, None, None)


def cross_attention(q, k, v, key_lengths=None, key_mask=None, scale=None):
    """softmax(scale * q k^T) v of queries q [B, Lq, H, D] over an encoder's states k, v [B, Lk, Hkv, D], as [B, Lq, H, D].

    Float32 or bf16, any strides (slices of a packed projection, expanded tensors); Hkv divides H, and head h reads state head h // (H // Hkv); D up to 128; scale 1 / sqrt(D) by default.
    key_lengths [B]: states at and behind it are not read; key_mask [B, Lk]: nor those where it is False.  What k and v hold there has no effect, not-a-number
    included, and their gradients are zero; a query without any state gives zeros.  Gradients are the same bits every time, whichever of them are asked for."""
    if ops._native is not None and q.is_cuda:
        dev = ops._current_device()
        got = ops._native.attention(q, k, v, key_lengths, key_mask, scale, dev, ops._raw_stream(dev))
        if got is not None:
            return ops._checked(got, "fovi_attention_forward")
    _no_tangents("cross_attention", q, k, v)
    if _wants_grad(q, k, v):
        return _AttentionFunction.apply(q, k, v, key_lengths, key_mask, scale)
    return ops.attention(q, k, v, key_lengths, key_mask, scale)


class _RmsNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        y, total, rstd = ops.rms_norm(x, weight, eps, residual, want_rstd=True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if total is None else total, weight, rstd)
        ctx.like = None if weight is None else (weight.dtype, weight.shape)
        return y if total is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, grad_total=None):
        t, weight, rstd = ctx.saved_tensors
        x_needs, w_needs, _, r_needs = ctx.needs_input_grad
        if grad is None:                                 # the norm's result was not used: the sum alone
            return (grad_total if x_needs else None), None, None, (grad_total if r_needs else None)
        dx, dw = ops.rms_norm_backward(t, grad, grad_total, weight, rstd, (x_needs or r_needs, w_needs))
        return (dx if x_needs else None), (None if dw is None else dw.to(ctx.like[0]).view(ctx.like[1])), None, (dx if r_needs else None)


def rms_norm(x, weight=None, eps=1e-6, residual=None):
    """Root-mean-square norm over the last axis: y = t / sqrt(mean(t^2) + eps) * weight of t = x, or with `residual` (x's shape and type) of t = x + residual as their type holds it:
    then (y, t) is returned, the same values as from the addition and the norm one after the other.  x [..., C] float32 or bf16; weight [C] or None.  Statistics, sums and the
    weight's gradient are float32; gradients are the same bits every time."""
    if ops._native is not None and x.is_cuda:
        dev = ops._current_device()
        got = ops._native.rms_norm(x, weight, eps, residual, dev, ops._raw_stream(dev))
        if got is not None:
            return ops._checked(got, "fovi_rms_norm_forward")
    _no_tangents("rms_norm", x, weight, residual)
    if _wants_grad(x, weight, residual):
        return _RmsNormFunction.apply(x, weight, eps, residual)
    y, total, _ = ops.rms_norm(x, weight, eps, residual)
    return y if total is None else (y, total)


def _no_gradient(name, *tensors):
    if _wants_grad(*tensors):
        raise NotImplementedError(f"{name}: what is held in 8 bits carries no gradient; call it under torch.no_grad(), or detach its tensors")


def rms_norm_int8(x, weight=None, eps=1e-6, residual=None):
    """rms_norm with its result in 8 bits for linear_int8: (q, scale), or (q, scale, t) with `residual`; y = q * scale to half a step.  q int8 [..., C], values of -127 .. 127 rounded
    from the unrounded y; scale float32 [...], max |y| / 127 of the row (at least the smallest normal number).  A row that holds infinity or not-a-number has one of them as its scale.
    No gradient."""
    if ops._native is not None and x.is_cuda:
        dev = ops._current_device()
        got = ops._native.rms_norm_int8(x, weight, eps, residual, dev, ops._raw_stream(dev))
        if got is not None:
            return ops._checked(got, "fovi_rms_norm_forward")
    _no_tangents("rms_norm_int8", x, weight, residual)
    _no_gradient("rms_norm_int8", x, weight, residual)
    q, scale, total = ops.rms_norm_int8(x, weight, eps, residual)
    return (q, scale) if total is None else (q, scale, total)


def quantize(x):
    """Rows of x [..., C] (float32 or bf16) in 8 bits with a scale each, as rms_norm_int8 gives them: tokens for linear_int8, or a weight [N, K] with a scale for each
    output channel.  No gradient."""
    if ops._native is not None and x.is_cuda:
        dev = ops._current_device()
        got = ops._native.quantize(x, dev, ops._raw_stream(dev))
        if got is not None:
            return ops._checked(got, "fovi_quantize_rows")
    _no_tangents("quantize", x)
    _no_gradient("quantize", x)
    return ops.quantize(x)


def linear_int8(q, scale, weight, weight_scale, bias=None, out_dtype=torch.bfloat16):
    """y = scale * weight_scale * (q weight^T) + bias: q int8 [..., K] with scale float32 [...], weight int8 [N, K] with weight_scale float32 [N], both as ``quantize`` gives them (or
    any other int8 tensors), bias [N] or None; K up to 131071.  The sums are exact; the result [..., N] is float32 or bf16.  No gradient."""
    if ops._native is not None and q.is_cuda:
        dev = ops._current_device()
        got = ops._native.linear_int8(q, scale, weight, weight_scale, bias, ops._DT.get(out_dtype, -2), dev, ops._raw_stream(dev))
        if got is not None:
            return ops._checked(got, "fovi_linear_int8")
    _no_tangents("linear_int8", scale, weight_scale, bias)
    _no_gradient("linear_int8", scale, weight_scale, bias)
    return ops.linear_int8(q, scale, weight, weight_scale, bias, out_dtype)


class _FeedForwardFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate_weight, up_weight, down_weight, gate_bias, up_bias, down_bias, activation):
        y, saved = ops.gated_feed_forward(x, gate_weight, up_weight, down_weight, gate_bias, up_bias, down_bias, activation, want_saved=True)
        ctx.save_for_backward(x, gate_weight, up_weight, down_weight, saved)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return ops.gated_feed_forward_backward(*ctx.saved_tensors, grad, ctx.activation, ctx.needs_input_grad[:7]) + (None,)


def gated_feed_forward(x, gate_weight, up_weight, down_weight, gate_bias=None, up_bias=None, down_bias=None, activation="silu"):
    """The gated feed-forward block of a transformer: (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd.  x [..., C], weights as torch's Linear has them (Wg, Wu [F, C], Wd [O, F]),
    biases [F], [F], [O] or None, all float32 or all bf16; activation "silu" or "gelu" (with the error function).  Differentiable in all tensors.  Sums are float32; with bf16 the
    hidden values, and in the backward pass their gradients, are rounded to bf16 between the products (few tokens without gradients: hidden values keep twice the bits).  Gradients are the same bits every time, whichever are asked for."""
    leaves = (x, gate_weight, up_weight, down_weight, gate_bias, up_bias, down_bias)
    if ops._native is not None and x.is_cuda and activation in ops.ACTIVATIONS:
        dev = ops._current_device()
        got = ops._native.gated_feed_forward(*leaves, ops.ACTIVATIONS[activation], dev, ops._raw_stream(dev))
        if got is not None:
            return ops._checked(got, "fovi_gated_ffn_forward")
    _no_tangents("gated_feed_forward", *leaves)
    if _wants_grad(*leaves):
        return _FeedForwardFunction.apply(*leaves, activation)
    return ops.gated_feed_forward(*leaves, activation)[0]


def check():
    """Synchronise the current stream and raise if an attention launch, or a product of linear_int8 or gated_feed_forward, on the current device since the last check, forward or
    backward, gave up on a bounded wait."""
    try:
        ops.attention_check()
    finally:
        ops.product_check()


# ------------------------------------------------------------------------------------------------------------ modules
class TokenNorm(nn.LayerNorm):
    """torch's LayerNorm over the last axis (same parameters, same state dict), on this package's kernels in both directions."""

    def __init__(self, dim, eps=1e-6, device="cuda", dtype=None):
        super().__init__(dim, eps=eps, device=device, dtype=dtype)

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)


class AxialRotary(nn.Module):
    """Rotary positions of tokens with `axes` coordinates.  The head's pairs are shared out evenly over the axes (`pairs_per_axis` says otherwise); pair j of an axis with n pairs
    has the frequency  unit * base^(-j / n), unit 2 pi for places in [-1, 1] (fovi/arch/knnvit.py:420-464).  `units`: one unit for each axis (1.0 for an
    axis that counts steps)."""

    def __init__(self, head_dim, axes=2, base=100.0, units=None, pairs_per_axis=None, pairing="halves", device="cuda"):
        super().__init__()
        if pairs_per_axis is None:
            pairs_per_axis = [head_dim // 2 // axes + (a < head_dim // 2 % axes) for a in range(axes)]
        units = [2 * math.pi] * len(pairs_per_axis) if units is None else units
        if len(units) != len(pairs_per_axis):
            raise ValueError(f"{len(units)} units for {len(pairs_per_axis)} axes")
        self.pairs_per_axis, self.pairing = tuple(int(n) for n in pairs_per_axis), pairing
        f = [u * base ** (-j / n) for u, n in zip(units, self.pairs_per_axis) for j in range(n)]
        self.register_buffer("frequencies", torch.tensor(f, dtype=torch.float32, device=device), persistent=False)

    def _apply(self, fn, recurse=True):      # stays float32 when the model is cast
        f = self.frequencies
        super()._apply(fn, recurse)
        if self.frequencies.dtype != torch.float32:
            self.frequencies = f.to(self.frequencies.device)
        return self

    def forward(self, x, positions, prefix=0):
        return rotary(x, positions, self.frequencies, self.pairs_per_axis, prefix, self.pairing)


class CrossAttention(nn.Module):
    """Multi-head attention of tokens x [B, Lq, dim] to states [B, Lk, state_dim]: projections (torch's Linear) around ``cross_attention``, with rotary positions on queries and
    states where `rotary` is given.  A program that asks the same states again keeps what ``project_states`` returns."""

    def __init__(self, dim, heads, kv_heads=None, state_dim=None, rotary=None, device="cuda", dtype=None):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if dim % heads or heads % kv_heads:
            raise ValueError(f"{dim} channels, {heads} heads, {kv_heads} state heads: each is to divide the one before")
        self.heads, self.kv_heads, self.head_dim, self.rotary = heads, kv_heads, dim // heads, rotary
        kw = dict(device=device, dtype=dtype)
        self.query = nn.Linear(dim, dim, **kw)
        self.key = nn.Linear(dim if state_dim is None else state_dim, kv_heads * self.head_dim, **kw)
        self.value = nn.Linear(dim if state_dim is None else state_dim, kv_heads * self.head_dim, **kw)
        self.out = nn.Linear(dim, dim, **kw)

    def project_states(self, states, positions=None, prefix=0):
        """states [B, Lk, state_dim] -> (k, v), each [B, Lk, kv_heads, head_dim], k turned by its positions."""
        shape = states.shape[:2] + (self.kv_heads, self.head_dim)
        k, v = self.key(states).view(shape), self.value(states).view(shape)
        return (k if positions is None else self.rotary(k, positions, prefix)), v

    def forward(self, x, kv, positions=None, prefix=0, key_lengths=None, key_mask=None):
        """x [B, Lq, dim]; kv: what project_states returned; positions: of x's tokens.  -> [B, Lq, dim]"""
        q = self.query(x).view(x.shape[:2] + (self.heads, self.head_dim))
        if positions is not None:
            q = self.rotary(q, positions, prefix)
        return self.out(cross_attention(q, *kv, key_lengths=key_lengths, key_mask=key_mask).flatten(2))


class TokenRMSNorm(nn.Module):
    """Root-mean-square norm with a weight (torch's RMSNorm by parameters and state dict).  Called with a residual it returns (norm of the sum, sum)."""

    def __init__(self, dim, eps=1e-6, device="cuda", dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, self.eps, residual)


class GatedFeedForward(nn.Module):
    """A block's gated feed-forward half: `gate`, `up` and `down` are torch's Linear by parameters and state dict; their values are taken in x's type, and both in autocast's where that
    is on."""

    def __init__(self, dim, hidden, activation="silu", bias=True, device="cuda", dtype=None):
        super().__init__()
        if activation not in ops.ACTIVATIONS:
            raise ValueError(f"activation is {activation!r}: 'silu' or 'gelu'")
        kw = dict(bias=bias, device=device, dtype=dtype)
        self.activation = activation
        self.gate, self.up, self.down = nn.Linear(dim, hidden, **kw), nn.Linear(dim, hidden, **kw), nn.Linear(hidden, dim, **kw)

    def forward(self, x):
        layers = (self.gate, self.up, self.down)
        if torch.is_autocast_enabled("cuda"):
            x = x.to(torch.get_autocast_dtype("cuda"))
        return gated_feed_forward(x, *(m.weight.to(x.dtype) for m in layers), *(None if m.bias is None else m.bias.to(x.dtype) for m in layers), activation=self.activation)


class Linear8(nn.Module):
    """A linear layer for serving in 8 bits, made from torch's Linear: its weight with a scale for each output channel, its input with one for each token.  Called with a tensor, which it
    quantises, or with the (q, scale) of rms_norm_int8 or quantize.  The result has `out_dtype`."""

    def __init__(self, linear, out_dtype=torch.bfloat16):
        super().__init__()
        self.out_dtype = out_dtype
        q, scale = quantize(linear.weight.detach())
        self.register_buffer("weight", q)
        self.register_buffer("weight_scale", scale)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().to(torch.float32, copy=True))

    def _apply(self, fn, recurse=True):      # scales and bias stay float32 when the model is cast
        kept = self.weight_scale, self.bias
        super()._apply(fn, recurse)
        for name, t in zip(("weight_scale", "bias"), kept):
            if t is not None and getattr(self, name).dtype != torch.float32:
                setattr(self, name, t.to(getattr(self, name).device))
        return self

    def forward(self, x, scale=None):
        q, scale = quantize(x) if scale is None else (x, scale)
        return linear_int8(q, scale, self.weight, self.weight_scale, self.bias, self.out_dtype)


class FixationReader(nn.Module):
    """Reads images out through several fixations: sensor -> foveated patch embedding -> the tokens of all fixations as one set of states, each with its place (the fixation's number,
    and the height and width in the image at which the token looks) -> learned queries, in `depth` pre-norm cross-attention blocks -> class scores.

    retina: RetinalTransform; embedding: KNNPatchEmbedding of `dim` channels that it feeds (not transposed).  feed_forward: hidden channels of a gated feed-forward half behind each
    block's attention, its norm fused with the addition of what the attention found; none by default."""

    def __init__(self, retina, embedding, dim, heads, n_classes, queries=1, depth=1, kv_heads=None, device="cuda", feed_forward=None):
        super().__init__()
        self.retina, self.embedding, self.dim = retina, embedding, dim
        self.rotary = AxialRotary(dim // heads, axes=3, units=[1.0, 2 * math.pi, 2 * math.pi], device=device)
        self.queries = nn.Parameter(torch.randn(queries, dim, device=device) * dim ** -0.5)
        self.state_norm = TokenNorm(dim, device=device)
        self.norms = nn.ModuleList([TokenNorm(dim, device=device) for _ in range(depth)])
        self.blocks = nn.ModuleList([CrossAttention(dim, heads, kv_heads, rotary=self.rotary, device=device) for _ in range(depth)])
        hidden = [] if feed_forward is None else [feed_forward] * depth
        self.feed_forward_norms = nn.ModuleList([TokenRMSNorm(dim, device=device) for _ in hidden])
        self.feed_forwards = nn.ModuleList([GatedFeedForward(dim, n, device=device) for n in hidden])
        self.norm = TokenNorm(dim, device=device)
        self.classifier = nn.Linear(dim, n_classes, device=device)

    def places(self, fix_rc, fix_hw, height, width):
        """float32 [B, F * tokens, 3]: fixation number, height and width (the image spans [-1, 1]) of every token.  fix_rc, fix_hw [B, F, 2] as the sensor takes them."""
        xy = self.embedding.out_coords.cartesian.to(device=fix_rc.device, dtype=torch.float32)
        reach = torch.stack([-xy[:, 1], xy[:, 0]], 1)                                            # (down, right) within the fixation, in its half sizes
        size = fix_hw.new_tensor([height, width])
        at = (2 * fix_rc - 1)[:, :, None] + reach * (fix_hw / size)[:, :, None]
        number = torch.arange(at.shape[1], device=at.device, dtype=at.dtype).view(1, -1, 1, 1).expand(at.shape[:3] + (1,))
        return torch.cat([number, at], -1).flatten(1, 2)

    def states(self, images, fix_loc, fixation_size=None):
        """images [B, 3, H, W], fix_loc [B, F, 2] -> (normed tokens of all fixations [B, F * tokens, dim], their places)."""
        fix_rc, fix_hw = self.retina.fixation_tensors(images, fix_loc, fixation_size)
        seen = self.retina(images, fix_rc, fix_hw)                                               # [B, F, 3, points]
        tokens = self.embedding(seen.flatten(0, 1))                                              # [B * F, tokens, dim]
        tokens = tokens.reshape(images.shape[0], -1, self.dim)
        return self.state_norm(tokens), self.places(fix_rc, fix_hw, *images.shape[2:])

    def read(self, states, places, key_lengths=None, key_mask=None):
        """Class scores [B, n_classes] from the states; key_lengths / key_mask: as for cross_attention."""
        x = self.queries.to(states.dtype).expand(states.shape[0], -1, -1)
        for i, (norm, block) in enumerate(zip(self.norms, self.blocks)):
            found = block(norm(x), block.project_states(states, places), key_lengths=key_lengths, key_mask=key_mask)
            if self.feed_forwards:
                normed, x = self.feed_forward_norms[i](found.to(x.dtype), residual=x)
                found = self.feed_forwards[i](normed)
            x = x + found
        return self.classifier(self.norm(x).mean(1))

    def forward(self, images, fix_loc, fixation_size=None, fixation_counts=None):
        """fixation_counts [B] (whole numbers): how many of an image's fixations count, all by default."""
        states, places = self.states(images, fix_loc, fixation_size)
        return self.read(states, places, None if fixation_counts is None else fixation_counts * len(self.embedding.out_coords))
