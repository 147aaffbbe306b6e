"""Operators on tokens, for what stands behind a foveated patch embedding: layer norm, rotary positions with several axes, and cross attention to an encoder's
states of another length, each with its gradients, on the library's own kernels.

In the reference they are torch calls inside its vision transformers (fovi/arch/vit.py:351-381: attention; fovi/arch/knnvit.py:420-464: rotary positions from the
tokens' sensor coordinates).  Here

* ``layer_norm`` / ``rotary`` / ``cross_attention`` are differentiable functions of tensors,
* ``TokenNorm`` / ``AxialRotary`` / ``CrossAttention`` the modules around them, and
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

__all__ = ["layer_norm", "rotary", "cross_attention", "TokenNorm", "AxialRotary", "CrossAttention", "FixationReader", "check"]


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


def check():
    """Synchronise the current stream and raise if an attention launch on the current device since the last check, forward or backward, gave up on a bounded wait."""
    ops.attention_check()


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


class FixationReader(nn.Module):
    """Reads images out through several fixations: sensor -> foveated patch embedding -> the tokens of all fixations as one set of states, each with its place (the fixation's number,
    and the height and width in the image at which the token looks) -> learned queries, in `depth` pre-norm cross-attention blocks -> class scores.

    retina: RetinalTransform; embedding: KNNPatchEmbedding of `dim` channels that it feeds (not transposed)."""

    def __init__(self, retina, embedding, dim, heads, n_classes, queries=1, depth=1, kv_heads=None, device="cuda"):
        super().__init__()
        self.retina, self.embedding, self.dim = retina, embedding, dim
        self.rotary = AxialRotary(dim // heads, axes=3, units=[1.0, 2 * math.pi, 2 * math.pi], device=device)
        self.queries = nn.Parameter(torch.randn(queries, dim, device=device) * dim ** -0.5)
        self.state_norm = TokenNorm(dim, device=device)
        self.norms = nn.ModuleList([TokenNorm(dim, device=device) for _ in range(depth)])
        self.blocks = nn.ModuleList([CrossAttention(dim, heads, kv_heads, rotary=self.rotary, device=device) for _ in range(depth)])
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
        for norm, block in zip(self.norms, self.blocks):
            x = x + block(norm(x), block.project_states(states, places), key_lengths=key_lengths, key_mask=key_mask)
        return self.classifier(self.norm(x).mean(1))

    def forward(self, images, fix_loc, fixation_size=None, fixation_counts=None):
        """fixation_counts [B] (whole numbers): how many of an image's fixations count, all by default."""
        states, places = self.states(images, fix_loc, fixation_size)
        return self.read(states, places, None if fixation_counts is None else fixation_counts * len(self.embedding.out_coords))
