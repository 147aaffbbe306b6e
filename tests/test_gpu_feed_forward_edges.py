"""GPU: the gated feed-forward block where its sizes and values are at an edge: workspaces, infinities, large gates, hooks on what it saves."""
import pytest
import torch

from oracle import block_oracle as oracle

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True, params=["native", "python"])
def launch_path(request, monkeypatch):
    """Every test with the native launch path (csrc/bind_tokens.h) and with the Python one."""
    from fovi_b200 import ops
    assert ops._native is not None
    if request.param == "python":
        monkeypatch.setattr(ops, "_native", None)


def _inputs(M, C, F, O, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    def n(*s, scale=1.0): return (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype)
    leaves = [n(M, C), n(F, C, scale=1.5 * C ** -0.5), n(F, C, scale=C ** -0.5), n(O, F, scale=F ** -0.5), n(F), n(F, scale=0.3), n(O, scale=0.3)]
    return leaves, n(M, O)


def _grads(leaves, dy, activation="silu"):
    from fovi_b200 import tokens
    for t in leaves:
        t.requires_grad_(True)
    y = tokens.gated_feed_forward(*leaves, activation=activation)
    return (y.detach(),) + torch.autograd.grad(y, leaves, dy)


# Hidden channels that leave 1 to 32 in their last 64: input gradients have one stage of k more in two pieces than in one.
LAST = [(885, 384, 1736, 384), (532, 768, 2080, 768), (233, 1280, 2968, 1280), (300, 64, 961, 64)]


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,C,F,O", LAST)
def test_gradients_of_uneven_hidden_channels(M, C, F, O, dtype):
    leaves, dy = _inputs(M, C, F, O, dtype, M)
    want = oracle.feed_forward(*[t.detach() for t in leaves], "silu", dy)
    for g, w in zip(_grads(leaves, dy), want, strict=True):
        oracle.near(g, w)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,C,F,O", LAST + [(40, 96, 1000, 96), (5, 384, 1021, 384)])
def test_nothing_is_written_behind_the_workspace(monkeypatch, M, C, F, O, dtype):
    from fovi_b200 import ops
    made, plain = [], ops._ffn_work

    def with_a_tail(*args):
        size, _ = plain(*args)
        made.append((size, torch.full((size + 65536,), 0xA5, dtype=torch.uint8, device="cuda")))
        return made[-1]
    monkeypatch.setattr(ops, "_ffn_work", with_a_tail)
    leaves, dy = _inputs(M, C, F, O, dtype, M)
    ops.gated_feed_forward(*leaves)
    _, saved = ops.gated_feed_forward(*leaves, want_saved=True)
    ops.gated_feed_forward_backward(*leaves[:4], saved, dy)
    for need in range(7):
        ops.gated_feed_forward_backward(*leaves[:4], saved, dy, need=[j == need for j in range(7)])
    assert len(made) == 10
    for size, work in made:
        assert (work[size:] == 0xA5).all()


@pytest.mark.autograd
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [1, 3, 300])
def test_slope_of_large_gates(M, dtype, activation):
    """The slope is one there, whatever the hidden channel beside it has for its gate, and the value the gate itself."""
    F = 128
    x = torch.ones(M, F, device="cuda", dtype=dtype)
    zero, eye = torch.zeros(F, F, device="cuda", dtype=dtype), torch.eye(F, device="cuda", dtype=dtype)
    wu = zero.clone()
    wu[:, 0] = 1
    large = 2.0 ** torch.arange(5, 5 + F // 2, device="cuda")                # 32 to 2^68
    gate = torch.stack([large, torch.linspace(-3, 5, F // 2, device="cuda")], 1).flatten().to(dtype)
    leaves = [x, zero, wu, eye, gate, None, None]
    for t in leaves[:5]:
        t.requires_grad_(True)
    from fovi_b200 import tokens
    y = tokens.gated_feed_forward(*leaves, activation=activation)
    dbg, = torch.autograd.grad(y, gate, torch.ones_like(y))
    g = gate.detach().double().requires_grad_(True)
    h = torch.nn.functional.silu(g) if activation == "silu" else torch.nn.functional.gelu(g)
    slope, = torch.autograd.grad(h.sum(), g)
    # bf16: a rounding each of h and y, and of dg and the bias's gradient, and the gate to 2^-16, which moves a slope of up to 1.13 by no more than 2^-16 |g| of the small ones; else float32's
    near = dict(rtol=2 ** -7 + 2 ** -11, atol=2 ** -12) if dtype is BF else dict(rtol=2 ** -19, atol=2 ** -20)
    torch.testing.assert_close(y.detach().double(), h.detach().expand(M, F), **near)
    torch.testing.assert_close(dbg.double(), M * slope, rtol=near["rtol"], atol=M * near["atol"])


def _by_definition(x, wg, wu, wd, bg, bu, bd, activation, dy):
    """Result and gradients in 64 bits, infinities and all, on the CPU."""
    x, wg, wu, wd, bg, bu, bd, dy = (t.detach().double().cpu() for t in (x, wg, wu, wd, bg, bu, bd, dy))
    g, u = x @ wg.T + bg, x @ wu.T + bu
    if activation == "silu":
        p = torch.sigmoid(g)
        slope = p * (1 + g * (1 - p))
    else:
        p = 0.5 * torch.erfc(-g / 2 ** 0.5)
        slope = p + g * torch.exp(-g * g / 2) / (2 * torch.pi) ** 0.5
    a = g * p
    h, dh = a * u, dy @ wd
    dg, du = dh * u * slope, dh * a
    return h @ wd.T + bd, dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ h, dg.sum(0), du.sum(0), dy.sum(0)


@pytest.mark.autograd
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("where", ["gate", "up"])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [1, 2, 300])
def test_infinity_in_the_gradients(M, dtype, value, where, activation):
    """A hidden channel that is infinite, or not a number: results and gradients are so exactly where the definition's are.  Tokens and the gradient of the result are positive, so that a
    gradient that sums infinities of one sign over the tokens stays infinite.  (The gate at -infinity is left out: the definition has 0 times infinity there.)"""
    if where == "gate" and value == -float("inf"):
        return
    leaves, dy = _inputs(M, 40, 100, 24, dtype, 3)
    leaves[0], dy = leaves[0].abs() + 0.125, dy.abs() + 0.125
    leaves[3] = leaves[3].abs() + 0.125
    leaves[4 if where == "gate" else 5][37] = value
    want = _by_definition(*leaves, activation, dy)
    infinite = 0
    for got, w in zip(_grads(leaves, dy, activation), want, strict=True):
        got, w = got.cpu().double(), w.to(dtype).double()
        assert torch.equal(got.isnan(), w.isnan())
        assert torch.equal(got.isinf(), w.isinf()) and torch.equal(got[w.isinf()], w[w.isinf()])
        infinite += w.isinf().sum().item()
    assert value != value or infinite >= 80


@pytest.mark.autograd
def test_the_largest_hidden_values():
    """Gates and up values near bf16's and float32's largest stay finite in what is kept for the backward pass."""
    from fovi_b200 import ops
    leaves, dy = _inputs(2, 8, 64, 8, BF, 5)
    x, wg, wu, wd = (torch.zeros_like(t) for t in leaves[:4])
    x[:, 0], wu[:, 0], wg[:, 1] = 1, 3.3895313892515355e38, 0
    x[:, 1], wu[:, 1] = 1, 1.3e36                                    # their sum: above bf16's largest value, below float32's
    wd[0, :] = 2.0 ** -126
    gate = torch.full((64,), 2.0, device="cuda", dtype=BF)
    _, saved = ops.gated_feed_forward(x, wg, wu, wd, gate, None, None, want_saved=True)
    grads = ops.gated_feed_forward_backward(x, wg, wu, wd, saved, torch.ones_like(dy))
    u, g = x.double() @ wu.double().T, gate.double()
    s = torch.sigmoid(g)
    dg = 2.0 ** -126 * u * s * (1 + g * (1 - s))
    # u kept to 2^-15, dg rounded to bf16, the sum of two tokens rounded once more
    torch.testing.assert_close(grads[4].double(), dg.sum(0), rtol=2 ** -7, atol=0)
