"""GPU: the persistent gradient kernels of bf16 cross attention where a block goes over several row tiles: more of them than SMs, with and without columns, long ones in front of short ones."""
import pytest
import torch

from oracle import token_oracle as oracle

pytestmark = [pytest.mark.gpu, pytest.mark.autograd]
BF = torch.bfloat16


def _inputs(B, Lq, Lk, H, Hkv, D, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return tuple(torch.randn(shape, generator=g, device="cuda").to(BF) for shape in ((B, Lq, H, D), (B, Lk, Hkv, D), (B, Lk, Hkv, D), (B, Lq, H, D)))


def _check(q, k, v, dy, per, key_lengths=None, key_mask=None):
    """Result and gradients, `per` samples at a time; states behind the longest of them are left out of the definition, and have gradients of zero."""
    from fovi_b200 import tokens
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = tokens.cross_attention(*leaves, key_lengths=key_lengths, key_mask=key_mask)
    got = (o.detach(),) + torch.autograd.grad(o, leaves, dy)
    tokens.check()
    for b in range(0, q.shape[0], per):
        at = slice(b, b + per)
        n = k.shape[1] if key_lengths is None else max(1, int(key_lengths[at].max()))
        want = oracle.attention(q[at], k[at, :n], v[at, :n], None if key_lengths is None else key_lengths[at], None if key_mask is None else key_mask[at, :n], dy=dy[at])
        for g, w in zip((got[0][at], got[1][at], got[2][at, :n], got[3][at, :n]), want):
            oracle.near(g, w)
        assert not got[2][at, n:].any() and not got[3][at, n:].any()


@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D", [(64, 33, 300, 20, 20, 64), (64, 140, 70, 20, 5, 64), (17, 257, 1030, 6, 6, 64), (40, 130, 200, 20, 20, 128), (24, 131, 701, 16, 4, 128),
                                             (90, 16, 261, 6, 1, 32)])
def test_several_row_tiles_a_block(B, Lq, Lk, H, Hkv, D):
    args = _inputs(B, Lq, Lk, H, Hkv, D, B + Lq)
    assert min((Lq + 127) // 128 * H, (Lk + 127) // 128 * Hkv) * B > 148
    g = torch.Generator(device="cuda").manual_seed(Lk)
    lengths = torch.randint(0, Lk + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    lengths[torch.rand(B, generator=g, device="cuda") < 0.3] = 0
    mask = torch.rand((B, Lk), generator=g, device="cuda") < 0.7
    mask[3] = False
    for kw in ({}, dict(key_lengths=lengths), dict(key_mask=mask), dict(key_lengths=lengths, key_mask=mask)):
        _check(*args, per=8, **kw)


@pytest.mark.parametrize("D", [64, 128])
def test_a_long_row_tile_in_front_of_short_ones(D):
    """A block's row tiles of very many columns, then several of one."""
    B, Lq, Lk, H = 40, 64, 12000, 20
    q, k, v, dy = _inputs(B, Lq, Lk, H, 1, D, 7)
    lengths = torch.ones(B, dtype=torch.int32, device="cuda")
    lengths[0] = lengths[15] = Lk
    lengths[3] = 0
    lengths[20:30] = 130
    for _ in range(5):
        _check(q, k, v, dy, per=1, key_lengths=lengths)
