"""GPU: the token operators' native launch path takes the plain forms, leaves the others to the Python path, and behaves in a graph as that one does."""
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


def _calls():
    from fovi_b200 import tokens
    x, w, b = torch.randn(40, 64, device="cuda"), torch.rand(64, device="cuda"), torch.rand(64, device="cuda")
    h = torch.randn(2, 20, 4, 64, device="cuda", dtype=BF)
    pos, f = torch.randn(20, 2, device="cuda"), torch.rand(32, device="cuda")
    lengths, mask = torch.tensor([20, 7], dtype=torch.int32, device="cuda"), torch.rand(2, 20, device="cuda") < 0.5
    plain = [(lambda: tokens.layer_norm(x, w, b)), (lambda: tokens.layer_norm(x.view(4, 10, 64))), (lambda: tokens.rotary(h, pos, f, (16, 16))),
             (lambda: tokens.rotary(h[:, 1:], pos.expand(2, -1, -1).contiguous()[:, 1:].contiguous(), f, (16, 16))), (lambda: tokens.cross_attention(h, h, h)),
             (lambda: tokens.cross_attention(h[:, :3], h, h, lengths, mask, 0.5)), (lambda: tokens.cross_attention(h.float(), h.float(), h.float()))]
    other = [(lambda: tokens.layer_norm(x.t())), (lambda: tokens.layer_norm(x, w.bfloat16())), (lambda: tokens.layer_norm(x[:0])),
             (lambda: tokens.rotary(h, pos, f, [16, 16])), (lambda: tokens.rotary(h.transpose(2, 3).contiguous().transpose(2, 3), pos, f, (16, 16))),
             (lambda: tokens.cross_attention(h, h, h, lengths.long())), (lambda: tokens.cross_attention(h, h.transpose(2, 3).contiguous().transpose(2, 3), h)),
             (lambda: tokens.cross_attention(h[:0], h[:0], h[:0]))]
    return plain, other


def test_which_calls_it_takes(counted):
    plain, other = _calls()
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
    x, w, b = (torch.randn(s, device="cuda") for s in ((300, 384), (384,), (384,)))
    h = torch.randn(2, 33, 4, 64, device="cuda", dtype=BF)
    pos, f = torch.randn(2, 32, 2, device="cuda"), torch.rand(32, device="cuda")

    def both(call, leaves):
        got = []
        for native in (ops._native, None):
            with monkeypatch.context() as m:
                m.setattr(ops, "_native", native)
                mine = [t.detach().requires_grad_(True) for t in leaves]
                y = call(*mine)
                got.append((y,) + torch.autograd.grad(y, mine, torch.ones_like(y).mul_(0.5)))
        for p, q in zip(*got):
            assert p.dtype == q.dtype and p.stride() == q.stride() and torch.equal(p, q)
    both(lambda x, w, b: tokens.layer_norm(x, w, b), (x, w, b))
    both(lambda h: tokens.rotary(h, pos, f, (16, 16), prefix=1), (h,))
    both(lambda q, k, v: tokens.cross_attention(q, k, v), (h, h, h))
    both(lambda q, k, v: tokens.cross_attention(q, k, v), (h.float(), h.float(), h.float()))


@pytest.mark.autograd
def test_in_a_graph(monkeypatch):
    """Names the gradient of the gradient as not built, notices inputs and results that were written to, gives its memory back, and adds up over several uses."""
    from fovi_b200 import ops, tokens
    for native in (ops._native, None):
        monkeypatch.setattr(ops, "_native", native)
        h = torch.randn(1, 5, 2, 64, device="cuda", requires_grad=True)
        x = torch.randn(6, 64, device="cuda", requires_grad=True)
        c = torch.randn(1, 7, 2, 64, device="cuda")
        pos, f = torch.randn(5, 2, device="cuda"), torch.rand(32, device="cuda")
        for call, leaf in ((lambda: tokens.layer_norm(x), x), (lambda: tokens.rotary(h, pos, f, (16, 16)), h), (lambda: tokens.cross_attention(h, c, c), h)):
            y = call()
            g, = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
            with pytest.raises(RuntimeError, match="differentiate"):
                g.sum().backward()
            y = call()
            y.sum().backward()
            with pytest.raises(RuntimeError, match="second time"):
                y.sum().backward()
            leaf.grad = None
            (call() + call()).sum().backward()
            twice, leaf.grad = leaf.grad, None
            call().sum().backward()
            assert torch.equal(twice, 2 * leaf.grad)
            leaf.grad = None
        a = x * 1.0
        y = tokens.layer_norm(a)
        a.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.sum().backward()
        y = tokens.cross_attention(h, h, h)
        z = y * 1.0
        y.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            z.sum().backward()


@pytest.mark.autograd
def test_backward_on_the_forwards_stream():
    from fovi_b200 import tokens
    side = torch.cuda.Stream()
    x = torch.randn(2000, 384, device="cuda", requires_grad=True)
    want, = torch.autograd.grad(tokens.layer_norm(x).square().sum(), x)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = tokens.layer_norm(x).square().sum()
    torch.cuda.current_stream().wait_stream(side)
    got, = torch.autograd.grad(y, x)
    assert torch.equal(got, want)
