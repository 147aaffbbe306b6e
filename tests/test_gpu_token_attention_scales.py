"""GPU: positive scales with masks, where bf16 calls go to the tensor cores (a scale of zero or below goes to the CUDA cores)."""
import pytest
import torch

from oracle import token_oracle as oracle

pytestmark = [pytest.mark.gpu, pytest.mark.autograd]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale", [1e-30, 0.02, 0.5, 4.0])
def test_scales_with_masks(scale, D, dtype):
    """A masked score loses and what the masked states hold stays out: single keys, whole tiles, all of a sample's, behind its length."""
    from fovi_b200 import tokens
    g = torch.Generator(device="cuda").manual_seed(23)
    q, k, v, dy = (torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((4, 66, 2, D), (4, 290, 1, D), (4, 290, 1, D), (4, 66, 2, D)))
    mask = torch.rand((4, 290), generator=g, device="cuda") < 0.6
    mask[1] = False
    mask[3, :128] = False
    kw = dict(key_mask=mask, key_lengths=torch.tensor([290, 290, 129, 200], dtype=torch.int32, device="cuda"), scale=scale)
    gone = ~mask | (torch.arange(290, device="cuda") >= kw["key_lengths"][:, None])
    clean = None
    for junk in (None, float("nan"), float("inf"), 3e38):
        leaves = [q] + [t if junk is None else t.masked_fill(gone[:, :, None, None], junk) for t in (k, v)]
        leaves = [t.detach().requires_grad_(True) for t in leaves]
        o = tokens.cross_attention(*leaves, **kw)
        got = (o.detach(),) + torch.autograd.grad(o, leaves, dy)
        if clean is None:
            clean = got
            for a, want in zip(got, oracle.attention(q, k, v, dy=dy, **kw)):
                oracle.near(a, want)
        assert all(torch.equal(a, b) for a, b in zip(got, clean))
    tokens.check()
