"""GPU: the gradients of cross attention have the same bits whichever of them are asked for."""
import itertools

import pytest
import torch

from oracle import token_oracle as oracle

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _inputs(B, Lq, Lk, H, Hkv, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(Lk + D)
    return tuple(torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((B, Lq, H, D), (B, Lk, Hkv, D), (B, Lk, Hkv, D), (B, Lq, H, D)))


# few keys, where a rounded result counts; shared state heads; more row tiles than SMs
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", [(4, 200, 2, 4, 4, 64), (4, 200, 6, 4, 4, 64), (3, 70, 300, 4, 2, 64), (2, 130, 129, 4, 4, 128), (2, 5, 90, 2, 1, 40), (2, 33, 77, 2, 2, 7),
                                   (20, 140, 300, 12, 12, 64), (20, 140, 300, 12, 3, 128)])
def test_any_choice_of_gradients(shape, dtype):
    from fovi_b200 import ops
    B, _, Lk = shape[:3]
    q, k, v, dy = _inputs(*shape, dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    lengths = torch.randint(0, Lk + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    lengths[0] = 0
    mask = torch.rand((B, Lk), generator=g, device="cuda") < 0.7
    for kw in ({}, dict(key_lengths=lengths), dict(key_lengths=lengths, key_mask=mask)):
        o, lse = ops.attention(q, k, v, want_lse=True, **kw)
        want = ops.attention_backward(q, k, v, o, dy, lse, **kw)
        for need in itertools.product((False, True), repeat=3):
            if any(need):
                for got, all_three, n in zip(ops.attention_backward(q, k, v, o, dy, lse, need=need, **kw), want, need):
                    assert torch.equal(got, all_three) if n else got is None
    ops.attention_check()


@pytest.mark.autograd
def test_frozen_queries_through_the_graph(monkeypatch):
    """Both launch paths; and with few keys the error of dk is as small as with dq (the bound is that of two roundings to bf16, with 1.1 for what is not rounded there)."""
    from fovi_b200 import ops, tokens
    q, k, v, dy = _inputs(4, 200, 3, 4, 4, 64, BF)
    exact = oracle.attention(q, k, v, dy=dy)[2][0]
    got = []
    for native, wants in itertools.product((ops._native, None), (True, False)):
        monkeypatch.setattr(ops, "_native", native)
        leaves = [t.detach().requires_grad_(True) for t in (k, v)]
        o = tokens.cross_attention(q.detach().requires_grad_(wants), *leaves)
        got.append(torch.autograd.grad(o, leaves, dy))
    for gk, gv in got:
        assert torch.equal(gk, got[0][0]) and torch.equal(gv, got[0][1])
        assert (gk.double() - exact).norm() <= 1.1 * 2 ** 0.5 * 2.0 ** -8 / 3 ** 0.5 * exact.norm()
