"""GPU: hooks on saved tensors see all that a token operator keeps for its backward pass, on both launch paths, and may move it."""
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.autograd]
BF, F32 = torch.bfloat16, torch.float32


def _r(*s, dtype=F32):
    return torch.randn(*s, device="cuda").to(dtype)


def _calls(dtype):
    """Name, function, leaves, whether its backward pass takes a part of its result."""
    from fovi_b200 import tokens
    x, w = _r(40, 64, dtype=dtype), _r(64)
    return [("layer_norm", tokens.layer_norm, (x, w, _r(64))),
            ("rms_norm", tokens.rms_norm, (x, w)),
            ("rms_norm with a residual", lambda x, w, r: tokens.rms_norm(x, w, residual=r), (x, w, _r(40, 64, dtype=dtype))),
            ("gated_feed_forward", tokens.gated_feed_forward, (x,) + tuple(_r(*s, dtype=dtype) for s in ((96, 64), (96, 64), (48, 96), (96,), (96,), (48,)))),
            ("cross_attention", tokens.cross_attention, tuple(_r(2, n, 4, 32, dtype=dtype) for n in (5, 9, 9)))]


def _graph(call, leaves):
    mine = [t.detach().requires_grad_(True) for t in leaves]
    y = call(*mine)
    return mine, y if isinstance(y, tuple) else (y,)


def _back(mine, ys):
    return torch.autograd.grad(ys, mine, [torch.full_like(y, 0.5) for y in ys])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("which", range(5))
def test_all_that_is_kept_passes_the_hooks(monkeypatch, which, dtype):
    from fovi_b200 import ops
    name, call, leaves = _calls(dtype)[which]
    native, seen, grads = ops._native, [], []
    for path in (native, None):
        monkeypatch.setattr(ops, "_native", path)
        mine, ys = _graph(call, leaves)
        grads.append(_back(mine, ys))
        packed = []

        def pack(t):
            packed.append((tuple(t.shape), t.dtype))
            return t.cpu()
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
            mine, ys = _graph(call, leaves)
        grads.append(_back(mine, ys))
        seen.append(sorted(packed, key=str))
    assert seen[0] == seen[1]
    for other in grads[1:]:
        assert all(torch.equal(p, q) for p, q in zip(grads[0], other, strict=True))


@pytest.mark.parametrize("path", ["native", "python"])
def test_a_feed_forward_blocks_memory_is_given_back(monkeypatch, path):
    """Under save_on_cpu the device keeps the leaves and the result; a checkpoint keeps no more, and has the same gradients."""
    from torch.utils.checkpoint import checkpoint
    from fovi_b200 import ops, tokens
    if path == "python":
        monkeypatch.setattr(ops, "_native", None)
    M, C, F = 4000, 128, 512
    leaves = [_r(*s, dtype=BF) for s in ((M, C), (F, C), (F, C), (C, F))]
    mine, ys = _graph(tokens.gated_feed_forward, leaves)
    want = _back(mine, ys)
    del mine, ys
    kept = ops.lib.fovi_gated_ffn_saved_bytes(1, M, F)
    for forms in (lambda *t: checkpoint(tokens.gated_feed_forward, *t, use_reentrant=False), None):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        if forms is None:
            with torch.autograd.graph.save_on_cpu():
                mine, ys = _graph(tokens.gated_feed_forward, leaves)
        else:
            mine, ys = _graph(forms, leaves)
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() - before < kept // 2              # the result is an eighth of what is kept
        assert all(torch.equal(p, q) for p, q in zip(want, _back(mine, ys), strict=True))
        del mine, ys


@pytest.mark.parametrize("which", range(5))
def test_what_a_hook_changed_is_refused(which):
    """Of what the operator itself made: the kernels would read behind a shorter one."""
    from fovi_b200 import ops
    assert ops._native is not None
    _, call, leaves = _calls(F32)[which]
    known = {tuple(t.shape) for t in leaves}
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t if tuple(t.shape) in known else t.flatten()[:-1].clone()):
        mine, ys = _graph(call, leaves)
    with pytest.raises(RuntimeError, match="saved-tensor hook"):
        _back(mine, ys)
