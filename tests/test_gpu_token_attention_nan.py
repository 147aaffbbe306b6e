"""GPU: cross attention with scores that are not a number, where the keys are read in one part and where they are cut into several that are joined."""
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.autograd]
BF, F32 = torch.bfloat16, torch.float32

# B, Lq, Lk, H, D: keys in one part and in several, of the kernels for few queries, of tiles on the CUDA cores (float32, and bf16 heads of 63 channels) and on the tensor cores
SHAPES = [(2, 70, 140, 2, 64), (7, 70, 300, 4, 64), (2, 70, 512, 2, 64), (1, 16, 2000, 2, 64), (1, 300, 4100, 2, 128), (2, 70, 512, 2, 63), (1, 3, 2000, 2, 64), (1, 1, 5000, 4, 128)]


def _inputs(B, Lq, Lk, H, D, dtype):
    g = torch.Generator(device="cuda").manual_seed(Lq + Lk)
    return tuple(torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((B, Lq, H, D), (B, Lk, H, D), (B, Lk, H, D), (B, Lq, H, D)))


def _run(q, k, v, dy, **kw):
    from fovi_b200 import tokens
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = tokens.cross_attention(*leaves, **kw)
    got = (o.detach(),) + torch.autograd.grad(o, leaves, dy)
    tokens.check()
    return got


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_query(shape, dtype):
    """Its row of the result is not a number, and nothing else; so are its dq, and dk and dv of the keys that its head reads."""
    q, k, v, dy = _inputs(*shape, dtype)
    q[-1, 0, 1, 5] = float("nan")
    o, dq, dk, dv = (torch.isnan(t) for t in _run(q, k, v, dy))
    for t in (o, dq):
        assert t[-1, 0, 1].all() and t.sum() == shape[4]
    for t in (dk, dv):
        assert t[-1, :, 1].all() and t.sum() == t[-1, :, 1].numel()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("where", ["first", "last", "all", "one"])
def test_states(shape, where, dtype):
    """Keys that are not a number, a whole part of them or one, are read: every row of their sample and head is not a number, the others are as without them."""
    B, Lq, Lk, H, D = shape
    q, k, v, dy = _inputs(*shape, dtype)
    want = _run(q, k, v, dy)
    at = dict(first=slice(0, Lk // 2), last=slice(Lk // 2, Lk), all=slice(0, Lk), one=slice(Lk - 3, Lk - 2))[where]
    k = k.clone()
    k[-1, at, 1] = float("nan")
    o, dq, dk, dv = _run(q, k, v, dy)
    assert torch.isnan(o[-1, :, 1]).all() and torch.isnan(dq[-1, :, 1]).all()
    for got, clean in zip((o, dq, dk, dv), want):
        others = torch.ones(B, H, dtype=torch.bool, device="cuda")
        others[-1, 1] = False
        assert torch.equal(got.transpose(1, 2)[others], clean.transpose(1, 2)[others])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_parts_without_a_key_stay_out(shape, dtype):
    """Parts whose keys are all masked, and hold what is not a number, have no effect; a sample without a key gives zeros, whatever its queries hold."""
    B, Lq, Lk, H, D = shape
    q, k, v, dy = _inputs(*shape, dtype)
    mask = torch.ones(B, Lk, dtype=torch.bool, device="cuda")
    mask[:, : Lk // 2] = False
    want = _run(q, k, v, dy, key_mask=mask)
    bad = ~mask[:, :, None, None]
    for a, b in zip(_run(q, k.masked_fill(bad, float("nan")), v.masked_fill(bad, float("nan")), dy, key_mask=mask), want):
        assert torch.equal(a, b) and torch.isfinite(a).all()
    q = torch.full_like(q, float("nan"))
    for t in _run(q, k, v, dy, key_lengths=torch.zeros(B, dtype=torch.int32, device="cuda")):
        assert not t.any()
