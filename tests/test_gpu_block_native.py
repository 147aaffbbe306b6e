"""GPU: the native launch path of a token block's operators takes the plain forms, leaves the others to the Python path, and behaves in a graph as that one does."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture
def counted(monkeypatch):
    """How many calls the native path took."""
    from fovi_b200 import ops
    native, taken = ops._native, []

    class Counting:
        def __getattr__(self, name):
            f = getattr(native, name)

            def call(*args):
                got = f(*args)
                taken.append(got is not None)
                return got
            return call
    monkeypatch.setattr(ops, "_native", Counting())
    return taken


def _block(dtype, M=40, C=64, F=96, O=48):
    return [torch.randn(*s, device="cuda").to(dtype) for s in ((M, C), (F, C), (F, C), (O, F), (F,), (F,), (O,))]


def test_which_calls_it_takes(counted):
    from fovi_b200 import tokens
    x, r, w = torch.randn(40, 64, device="cuda"), torch.randn(40, 64, device="cuda"), torch.rand(64, device="cuda")
    q, s = tokens.quantize(x)
    q3, s3 = tokens.quantize(x[:, :61].contiguous())
    leaves, plain32 = _block(BF), _block(torch.float32, C=61, F=33, O=5)
    counted.clear()
    plain = [lambda: tokens.rms_norm(x, w), lambda: tokens.rms_norm(x.view(4, 10, 64), residual=r.view(4, 10, 64)), lambda: tokens.rms_norm_int8(x, w, residual=r),
             lambda: tokens.rms_norm_int8(x[0]), lambda: tokens.quantize(x), lambda: tokens.linear_int8(q, s, q, s, s), lambda: tokens.linear_int8(q3, s3, q3, s3, out_dtype=torch.float32),
             lambda: tokens.linear_int8(q.view(4, 10, 64), s.view(4, 10), q, s), lambda: tokens.gated_feed_forward(*leaves), lambda: tokens.gated_feed_forward(*leaves[:4]),
             lambda: tokens.gated_feed_forward(*plain32, activation="gelu"), lambda: tokens.gated_feed_forward(*_block(BF, C=61)), lambda: tokens.gated_feed_forward(*_block(BF, F=33, O=5))]
    other = [lambda: tokens.rms_norm(x.t()), lambda: tokens.rms_norm(x, w.to(BF)), lambda: tokens.rms_norm(x[:0]), lambda: tokens.rms_norm(x, w, residual=r.t().contiguous().t()),
             lambda: tokens.rms_norm_int8(x[:, ::2]), lambda: tokens.quantize(x[:, ::2]), lambda: tokens.linear_int8(q[:, 1:], s, q[:, 1:].contiguous(), s),
             lambda: tokens.linear_int8(q, s, q, s, s.to(BF)), lambda: tokens.linear_int8(q[:0], s[:0], q, s), lambda: tokens.gated_feed_forward(leaves[0][:, ::2], *_block(BF, C=32)[1:]),
             lambda: tokens.gated_feed_forward(leaves[0][:0], *leaves[1:])]
    for call in plain:
        call()
    assert counted == [True] * len(plain)
    counted.clear()
    for call in other:
        call()
    assert counted == [False] * len(other)


@pytest.mark.autograd
def test_gradients_are_the_same_bits(monkeypatch):
    from fovi_b200 import ops, tokens

    def both(call, leaves, some=None):
        got = []
        for native in (ops._native, None):
            with monkeypatch.context() as m:
                m.setattr(ops, "_native", native)
                mine = [t.detach().requires_grad_(some is None or i in some) for i, t in enumerate(leaves)]
                y = call(*mine)
                y = y if isinstance(y, tuple) else (y,)
                got.append(y + torch.autograd.grad(y, [t for t in mine if t.requires_grad], [torch.ones_like(o).mul_(0.5) for o in y]))
        for p, q in zip(*got, strict=True):
            assert p.dtype == q.dtype and p.stride() == q.stride() and torch.equal(p, q)
    x, r, w = torch.randn(300, 384, device="cuda"), torch.randn(300, 384, device="cuda"), torch.randn(384, device="cuda")
    for dtype in (torch.float32, BF):
        both(lambda x, w: tokens.rms_norm(x, w), (x.to(dtype), w))
        both(lambda x, r, w: tokens.rms_norm(x, w, residual=r), (x.to(dtype), r.to(dtype), w))
        both(lambda x, r, w: tokens.rms_norm(x, w, residual=r), (x.to(dtype), r.to(dtype), w), (1,))
        leaves = _block(dtype)
        both(lambda *t: tokens.gated_feed_forward(*t), leaves)
        both(lambda *t: tokens.gated_feed_forward(*t, activation="gelu"), leaves[:4])
        for i in range(7):
            both(lambda *t: tokens.gated_feed_forward(*t), leaves, (i,))


@pytest.mark.autograd
def test_in_a_graph(monkeypatch):
    """Names the gradient of the gradient as not built, notices inputs and results that were written to, gives its memory back, and adds up over several uses."""
    from fovi_b200 import ops, tokens
    for native in (ops._native, None):
        monkeypatch.setattr(ops, "_native", native)
        x, r = (torch.randn(6, 64, device="cuda", requires_grad=True) for _ in range(2))
        leaves = _block(torch.float32)[1:]
        for call, leaf in ((lambda: tokens.rms_norm(x), x), (lambda: sum(tokens.rms_norm(x, residual=r)), r), (lambda: tokens.gated_feed_forward(x, *leaves), x)):
            y = call()
            g, = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
            with pytest.raises(RuntimeError, match="differentiate"):
                g.sum().backward()
            y = call()
            y.sum().backward()
            with pytest.raises(RuntimeError, match="second time"):
                y.sum().backward()
            x.grad = r.grad = None
            (call() + call()).sum().backward()
            twice, x.grad, r.grad = leaf.grad, None, None
            call().sum().backward()
            assert torch.equal(twice, 2 * leaf.grad)
            x.grad = r.grad = None
        # a leaf's own gradient, although both inputs are given one tensor's values
        y, total = tokens.rms_norm(x, residual=r)
        (y.sum() + total.sum()).backward()
        x.grad.add_(1)
        assert not torch.equal(x.grad, r.grad)
        x.grad = r.grad = None
        a = x * 1.0
        y = tokens.rms_norm(a)
        a.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.sum().backward()
        y, total = tokens.rms_norm(x, residual=r)
        z = total * 1.0
        total.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            (z.sum() + y.sum()).backward()
        a = x * 1.0
        y = tokens.gated_feed_forward(a, *leaves)
        a.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.sum().backward()


@pytest.mark.autograd
def test_tangents_are_refused(monkeypatch):
    from torch.autograd import forward_ad
    from fovi_b200 import ops, tokens
    x, r, w = torch.randn(6, 64, device="cuda"), torch.randn(6, 64, device="cuda"), torch.rand(64, device="cuda")
    q, s = tokens.quantize(x)
    calls = [("rms_norm", lambda x, w, r: tokens.rms_norm(x, w, residual=r), (x, w, r)), ("rms_norm_int8", lambda x, w, r: tokens.rms_norm_int8(x, w, residual=r), (x, w, r)),
             ("quantize", tokens.quantize, (x,)), ("linear_int8", lambda a, b, c: tokens.linear_int8(q, a, q, b, c), (s, s.clone(), s.clone())),
             ("gated_feed_forward", tokens.gated_feed_forward, _block(torch.float32))]
    for native in (ops._native, None):
        monkeypatch.setattr(ops, "_native", native)
        for name, call, args in calls:
            for i in range(len(args)):
                with forward_ad.dual_level():
                    mine = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
                    with pytest.raises(NotImplementedError, match=f"{name}: forward-mode"):
                        call(*mine)
            with pytest.raises((RuntimeError, NotImplementedError)):
                torch.func.vmap(lambda x: call(x, *args[1:]))(torch.stack([args[0], args[0]]))


@pytest.mark.autograd
def test_backward_on_the_forwards_stream():
    from fovi_b200 import tokens
    side = torch.cuda.Stream()
    leaves = _block(BF, M=2000)
    x = leaves[0].requires_grad_(True)

    def loss():
        return tokens.gated_feed_forward(tokens.rms_norm(x), *leaves[1:]).float().square().sum()
    want, = torch.autograd.grad(loss(), x)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = loss()
    torch.cuda.current_stream().wait_stream(side)
    got, = torch.autograd.grad(y, x)
    assert torch.equal(got, want)
