"""GPU: the token operators have no forward-mode derivatives and no batching rules, and say so: a result without its tangent would read as a derivative of zero."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["native", "python"])
def launch_path(request, monkeypatch):
    from fovi_b200 import ops
    assert ops._native is not None
    if request.param == "python":
        monkeypatch.setattr(ops, "_native", None)


def _calls(dtype):
    """Name, function and tensors of each operator."""
    from fovi_b200 import tokens
    x, w, b = torch.randn(6, 64, device="cuda").to(dtype), torch.rand(64, device="cuda"), torch.rand(64, device="cuda")
    h, c = torch.randn(2, 5, 2, 64, device="cuda").to(dtype), torch.randn(2, 7, 2, 64, device="cuda").to(dtype)
    return [("layer_norm", tokens.layer_norm, (x, w, b)), ("rotary", lambda x, p, f: tokens.rotary(x, p, f, (16, 16)), (h, torch.randn(5, 2, device="cuda"), torch.rand(32, device="cuda"))),
            ("cross_attention", tokens.cross_attention, (h, c, c.flip(1)))]


@pytest.mark.autograd
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_tangent_is_refused(dtype, graph):
    """On each of the tensors, whether or not gradients are asked for too."""
    for name, call, args in _calls(dtype):
        for i in range(len(args)):
            with forward_ad.dual_level():
                mine = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
                if graph:
                    mine[0] = mine[0].requires_grad_(True)
                with pytest.raises(NotImplementedError, match=f"{name}: forward-mode"):
                    call(*mine)


def test_a_level_without_tangents_changes_nothing():
    for _, call, args in _calls(torch.float32):
        want = call(*args)
        with forward_ad.dual_level():
            duals = [forward_ad.make_dual(t, torch.ones_like(t)) for t in args]
            assert torch.equal(call(*args), want)
            assert torch.equal(call(*(forward_ad.unpack_dual(t).primal for t in duals)), want)
        assert torch.equal(call(*(t.clone() for t in args)), want)


@pytest.mark.autograd
def test_function_transforms_are_refused():
    for _, call, args in _calls(torch.float32):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(lambda x: call(x, *args[1:]), (args[0],), (torch.ones_like(args[0]),))
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.vmap(lambda x: call(x, *args[1:]))(torch.stack([args[0], args[0]]))
