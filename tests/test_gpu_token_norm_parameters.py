"""GPU: layer norm's weight and bias are C values in any shape, and their gradients have that shape and type."""
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.autograd]


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,bias_shape", [((64,), (64,)), ((1, 64), (64,)), ((64, 1), (1, 1, 64)), ((64,), None), (None, (1, 64))])
def test_gradients_have_the_parameters_shapes(shape, bias_shape, dtype, native, monkeypatch):
    from fovi_b200 import ops, tokens
    if not native:
        monkeypatch.setattr(ops, "_native", None)
    x, dy = torch.randn(40, 64, device="cuda"), torch.randn(40, 64, device="cuda")
    flat = [torch.rand(64, device="cuda").to(dtype) for _ in range(2)]
    shaped = [None if s is None else t.reshape(s).requires_grad_(True) for s, t in zip((shape, bias_shape), flat)]
    plain = [None if s is None else t.detach().requires_grad_(True) for s, t in zip((shape, bias_shape), flat)]
    y, want = tokens.layer_norm(x, *shaped), tokens.layer_norm(x, *plain)
    assert torch.equal(y, want)
    y.backward(dy)
    want.backward(dy)
    for p, f in zip(shaped, plain):
        if p is not None:
            assert p.grad.shape == p.shape and p.grad.dtype is p.dtype and torch.equal(p.grad.reshape(-1), f.grad)
