"""GPU: the gated feed-forward block and its gradients against the definition in 64 bits."""
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


def _inputs(M, C, F, O, dtype, seed, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    def n(*s, scale=1.0): return (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype)
    x, wg, wu, wd = n(M, C), n(F, C, scale=1.5 * C ** -0.5), n(F, C, scale=C ** -0.5), n(O, F, scale=F ** -0.5)
    biases = [n(F), n(F, scale=0.3), n(O, scale=0.3)] if bias else [None] * 3
    return [x, wg, wu, wd] + biases, n(M, O)


def _grads(leaves, dy, activation):
    from fovi_b200 import tokens
    for t in leaves:
        if t is not None:
            t.requires_grad_(True)
    y = tokens.gated_feed_forward(*leaves, activation=activation)
    return (y,) + torch.autograd.grad(y, [t for t in leaves if t is not None], dy)


def _wanted(leaves, dy, activation):
    plain = [None if t is None else t.detach() for t in leaves]
    want = oracle.feed_forward(*plain, activation, dy)
    return want[:1] + [w for w, t in zip(want[1:], leaves) if t is not None]


SIZES = [(1, 8, 8, 8), (1, 384, 1024, 384), (1, 1280, 5120, 1280), (3, 5, 7, 2), (1, 1, 1, 1), (8, 384, 1024, 384), (9, 40, 72, 24), (16, 100, 260, 100), (31, 384, 1021, 390), (33, 64, 64, 64),
         (65, 96, 130, 33), (65, 1280, 3416, 1280), (127, 136, 344, 136), (128, 128, 256, 128), (129, 384, 341, 384), (257, 1280, 24, 80), (300, 390, 520, 130), (700, 64, 1000, 64),
         (2500, 48, 16, 40), (4200, 384, 1024, 384), (48, 384, 1024, 384), (200, 96, 256, 100), (1000, 40, 64, 48), (1030, 24, 40, 16), (150, 301, 777, 203), (1028, 384, 1021, 384), (513, 768, 2048, 768)]


@pytest.mark.autograd
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,C,F,O", SIZES)
def test_forward_and_gradients(M, C, F, O, dtype, activation):
    from fovi_b200 import tokens
    bias = (M + C) % 2 == 1 or activation == "gelu"
    leaves, dy = _inputs(M, C, F, O, dtype, M + C + F, bias)
    got = _grads(leaves, dy, activation)
    assert got[0].dtype is dtype and got[0].is_contiguous()
    for g, want in zip(got, _wanted(leaves, dy, activation), strict=True):
        assert g.dtype is dtype and g.is_contiguous()
        oracle.near(g.detach(), want)
    with torch.no_grad():
        oracle.near(tokens.gated_feed_forward(*leaves, activation=activation), oracle.feed_forward(*leaves, activation)[0])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,C,F,O", [(5, 96, 200, 96), (400, 96, 200, 96), (150, 31, 77, 45)])
def test_gradients_one_by_one_are_the_same_bits(M, C, F, O, dtype):
    from fovi_b200 import ops
    leaves, dy = _inputs(M, C, F, O, dtype, 4)
    _, saved = ops.gated_feed_forward(*leaves, want_saved=True)
    every = ops.gated_feed_forward_backward(*leaves[:4], saved, dy)
    for _ in range(2):
        assert all(torch.equal(p, q) for p, q in zip(every, ops.gated_feed_forward_backward(*leaves[:4], saved, dy)))
    for i in range(7):
        got = ops.gated_feed_forward_backward(*leaves[:4], saved, dy, need=[j == i for j in range(7)])
        assert torch.equal(got[i], every[i]) and all(got[j] is None for j in range(7) if j != i)


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [4, 200])
def test_strides_and_shapes(M, dtype):
    """Slices on 16-byte boundaries and off them, transposed weights, an expanded input and gradient, several leading axes."""
    from fovi_b200 import tokens
    C, F = 64, 120

    def check(leaves, dy):
        for g, want in zip(_grads(leaves, dy, "silu"), _wanted(leaves, dy, "silu"), strict=True):
            oracle.near(g.detach(), want)
    for lo in (0, 8, 1):
        leaves, dy = _inputs(M, C + 16, F + 16, C + 16, dtype, lo)
        x, wg, wu, wd, bg, bu, bd = leaves
        check([t.detach() for t in (x[:, lo:lo + C], wg[lo:lo + F, lo:lo + C], wu[:F, lo:lo + C], wd[:C, lo:lo + F], bg[lo:lo + F], bu[:F], bd[1:C + 1])], dy[:, lo:lo + C])
    leaves, dy = _inputs(M, C, F, C, dtype, 7)
    x, wg, wu, wd = leaves[:4]
    check([x.t().contiguous().t(), wg.t().contiguous().t(), wu, wd.t().contiguous().t()] + leaves[4:], dy.t().contiguous().t())
    check([x[:1].detach().expand(M, C)] + [t.detach() for t in leaves[1:]], dy[:1].expand(M, C))
    with torch.no_grad():
        y = tokens.gated_feed_forward(*leaves)
        assert torch.equal(tokens.gated_feed_forward(x.view(2, 1, M // 2, C), *leaves[1:]), y.view(2, 1, M // 2, C))
        one = tokens.gated_feed_forward(x[0], *leaves[1:])
        assert one.shape == (C,) and torch.equal(one, tokens.gated_feed_forward(x[:1], *leaves[1:])[0])


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
def test_no_tokens(dtype):
    leaves, dy = _inputs(0, 24, 40, 16, dtype, 1)
    y, dx, *rest = _grads(leaves, dy, "silu")
    assert y.shape == (0, 16) and dx.shape == (0, 24) and not any(t.any() for t in rest)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [3, 300])
def test_far_values(M, dtype):
    """Gates whose exponentials leave the range of float32 on either side."""
    from fovi_b200 import tokens
    leaves, _ = _inputs(M, 64, 96, 64, dtype, 2)
    leaves[4] = (torch.arange(96, device="cuda") * 4.0 - 190).to(dtype)
    for activation in ("silu", "gelu"):
        oracle.near(tokens.gated_feed_forward(*leaves, activation=activation), oracle.feed_forward(*leaves, activation)[0])
    x = leaves[0]
    x[1, 5] = float("nan")
    y = tokens.gated_feed_forward(*leaves)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2:]).all()


@pytest.mark.autograd
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_gradient_against_differences(activation):
    """Central differences of the kernel's own forward pass along a random direction; the difference between two step sizes bounds the truncation."""
    from fovi_b200 import tokens
    leaves, dy = _inputs(6, 20, 28, 12, F32, 21)
    g = torch.Generator(device="cuda").manual_seed(1)
    dirs = [torch.randn(t.shape, generator=g, device="cuda") * 0.3 for t in leaves]
    grads = _grads(leaves, dy, activation)[1:]
    with torch.no_grad():
        size = oracle.feed_forward(*leaves, activation)[0][1].max().item()
        for i in range(7):
            def loss(h):
                args = [t + h * d if j == i else t for j, (t, d) in enumerate(zip(leaves, dirs))]
                return (tokens.gated_feed_forward(*args, activation=activation).double() * dy.double()).sum().item()
            near, far = ((loss(h) - loss(-h)) / (2 * h) for h in (2.0 ** -7, 2.0 ** -6))
            rounding = 4 * size * dy.double().abs().sum().item() / 2.0 ** -7
            assert abs((grads[i].double() * dirs[i].double()).sum().item() - near) <= abs(near - far) + rounding


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
def test_module(dtype):
    """Parameters under torch's names, in their own type; a stream that is not the default one."""
    from fovi_b200.tokens import GatedFeedForward
    m = GatedFeedForward(48, 80, activation="gelu")
    assert sorted(m.state_dict()) == sorted(f"{a}.{b}" for a in ("gate", "up", "down") for b in ("weight", "bias"))
    assert not any(k.endswith("bias") for k in GatedFeedForward(48, 80, bias=False).state_dict())
    x, dy = torch.randn(2, 30, 48, device="cuda").to(dtype).requires_grad_(True), torch.randn(2, 30, 48, device="cuda").to(dtype)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = m(x)
        y.backward(dy)
    torch.cuda.current_stream().wait_stream(stream)
    layers = (m.gate, m.up, m.down)
    args = [x.detach().flatten(0, 1)] + [t.weight.detach().to(dtype) for t in layers] + [t.bias.detach().to(dtype) for t in layers]
    want = oracle.feed_forward(*args, "gelu", dy.flatten(0, 1))
    got = [y.flatten(0, 1), x.grad.flatten(0, 1)] + [t.weight.grad for t in layers] + [t.bias.grad for t in layers]
    for g, w in zip(got, want, strict=True):
        oracle.near(g.detach(), w)
    assert all(p.grad.dtype is F32 for p in m.parameters())


@pytest.mark.autograd
def test_refusals():
    from fovi_b200 import ops, tokens
    leaves, dy = _inputs(4, 16, 24, 8, F32, 1)
    def refused(error, words, **change):
        args = {**dict(zip("x wg wu wd bg bu bd".split(), leaves)), **change}
        with pytest.raises(error, match=words):
            tokens.gated_feed_forward(*(args[k] for k in "x wg wu wd bg bu bd".split()), **({"activation": args["act"]} if "act" in args else {}))
    x, wg, wu, wd, bg, bu, bd = leaves
    for name, t in zip("x wg wu wd bg bu bd".split(), leaves):
        refused(ValueError, "CUDA", **{name: t.cpu()})
        refused(TypeError, "same type", **{name: t.bfloat16()})
    refused(TypeError, "dtype", **dict(zip("x wg wu wd bg bu bd".split(), [t.half() for t in leaves])))
    refused(ValueError, "wanted", x=x[:, :8])
    refused(ValueError, "wanted", wu=wu[:8])
    refused(ValueError, "wanted", wd=wd[:, :8])
    refused(ValueError, "wanted", wg=wg[0])
    refused(ValueError, "wanted", wd=wd[:0], bd=None)
    refused(ValueError, "gate bias", bg=bg[:4])
    refused(ValueError, "up bias", bu=bu[:, None])
    refused(ValueError, "down bias", bd=bg)
    refused(ValueError, "activation", act="relu")
    with pytest.raises(ValueError, match="activation"):
        tokens.GatedFeedForward(8, 8, activation="relu")
    _, saved = ops.gated_feed_forward(*leaves, want_saved=True)
    with pytest.raises(ValueError, match="gradient has the shape"):
        ops.gated_feed_forward_backward(x, wg, wu, wd, saved, dy[:, :4])
    with pytest.raises(ValueError, match="saved"):
        ops.gated_feed_forward_backward(x, wg, wu, wd, saved[:-1], dy)
    y = tokens.gated_feed_forward(x.requires_grad_(True), *leaves[1:])
    first, = torch.autograd.grad(y, x, torch.ones_like(y, requires_grad=True), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), x)


@pytest.mark.autograd
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [4, 16, 300])
def test_gates_far_from_zero(M, dtype, activation):
    """Gates from -1e20 to 1e3 with an up value of one, taken out unchanged: below -40 the value and the slope are zeros."""
    F = 64
    x = torch.zeros(M, F, device="cuda", dtype=dtype)
    x[:, 0], x[:, 1] = 1e10, 1
    gates = torch.tensor([-1e10, -1e3, -1e-5, -1e-8, -4e-9, -1e-9, 1e-10, 1e-7], device="cuda").repeat(F // 8)
    wg, wu = torch.zeros(F, F, device="cuda", dtype=dtype), torch.zeros(F, F, device="cuda", dtype=dtype)
    wg[:, 0], wu[:, 1] = gates.to(dtype), 1
    leaves = [x, wg, wu, torch.eye(F, device="cuda", dtype=dtype)] + [None] * 3
    with torch.no_grad():
        from fovi_b200 import tokens
        few = tokens.gated_feed_forward(*leaves, activation=activation)
    y, _, dwg, dwu, _ = _grads(leaves, torch.ones(M, F, device="cuda", dtype=dtype), activation)
    g = (x[0, 0].detach().double() * wg.detach()[:, 0].double()).requires_grad_(True)
    h = torch.nn.functional.silu(g) if activation == "silu" else torch.nn.functional.gelu(g)
    slope, = torch.autograd.grad(h.sum(), g)
    # Two roundings each, of h and y or of dg or du and the weight's gradient; the gate is kept to 2^-17 of its value, which moves a value and a slope by no more than 41 (|g| where they
    # are not zeros) times that.  The rest is zero to 1e-16 (value and slope below -41: 41.6 x 2^-60), a gradient's to that times the rows.
    near = dict(rtol=2 ** -7 + 2 ** -11, atol=1e-16)
    for got in (few, y):
        torch.testing.assert_close(got.double(), h.detach().expand(M, F), **near)
    torch.testing.assert_close(dwg[:, 1].double(), M * slope, rtol=near["rtol"], atol=M * 1e-16)
    torch.testing.assert_close(dwu[:, 1].double(), M * h.detach(), rtol=near["rtol"], atol=M * 1e-16)


def _in_64_bits(leaves, activation):
    x, wg, wu, wd, bg, bu, bd = (t.detach().double() for t in leaves)
    g, u = x @ wg.T + bg, x @ wu.T + bu
    h = (torch.nn.functional.silu(g) if activation == "silu" else torch.nn.functional.gelu(g)) * u
    return g, u, h, wd, bd


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("M,C,F,O", [(1, 1280, 5120, 1280), (3, 115, 312, 115), (1, 1280, 18, 1280), (8, 118, 320, 118), (16, 40, 24, 40), (40, 96, 256, 96)])
def test_few_tokens_are_rounded_once(M, C, F, O, activation):
    """Without gradients few tokens' hidden values keep 16 bits and more: what is left is the result's own rounding."""
    from fovi_b200 import tokens
    leaves, _ = _inputs(M, C, F, O, BF, 3 * M + F)
    with torch.no_grad():
        y = tokens.gated_feed_forward(*leaves, activation=activation).double()
    _, _, h, wd, bd = _in_64_bits(leaves, activation)
    # Half a step of the result; a hidden value's parts leave 2^-17 of it, its logistic function (approximate exponential and quotient) 2^-20; and float32 sums: of F products for the
    # result, of C for g and u, which an activation's slope of up to 1.13 hands on times u, and act(g), at most |g|, times u's.
    x, wg, wu, _, bg, bu, _ = (t.detach().double().abs() for t in leaves)
    size, sum_g, sum_u = h.abs() @ wd.abs().T + bd.abs(), x @ wg.T + bg, x @ wu.T + bu
    hidden = 2.0 ** -16 * h.abs() + 2.2 * C * 2.0 ** -24 * sum_g * sum_u
    assert ((y - (h @ wd.T + bd)).abs() <= 2 ** -8 * (h @ wd.T + bd).abs() + hidden @ wd.abs().T + F * 2.0 ** -24 * size).all()


@pytest.mark.autograd
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("M,C,F", [(2, 384, 1536), (77, 22, 88), (314, 1280, 14), (525, 129, 344), (5000, 96, 79)])
def test_gradients_of_biases_are_rounded_once(M, C, F, activation):
    leaves, dy = _inputs(M, C, F, C, BF, M + F)
    _, _, _, _, _, dbg, dbu, dbd = _grads(leaves, dy, activation)
    g, u, h, wd, _ = _in_64_bits(leaves, activation)
    g.requires_grad_(True)
    a = torch.nn.functional.silu(g) if activation == "silu" else torch.nn.functional.gelu(g)
    slope, = torch.autograd.grad(a.sum(), g)
    a, dh = a.detach(), dy.double() @ wd
    # Half a step of the result; g and u are kept to 2^-17, which a slope (its own slope is at most 0.8, |g| up to 8 or the slope is flat) takes as 2^-14; sums of C and M products in float32.
    far = 2 ** -13 + (C + M) * 2 ** -24
    size = dy.double().abs() @ wd.abs()
    for got, each, most in ((dbg, dh * u * slope, size * (u.abs() + 1)), (dbu, dh * a, size * (a.abs() + 1))):
        want = each.sum(0)
        assert ((got.double() - want).abs() <= 2 ** -8 * want.abs() + far * most.sum(0)).all()
    torch.testing.assert_close(dbd.double(), dy.double().sum(0), rtol=2 ** -8, atol=M * 2 ** -24 * dy.abs().sum(0).max().item())


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [4, 300])
def test_infinity_stays_infinity(M, dtype, activation):
    """Weights above zero: a token with infinity in it has an infinite result, with and without what a backward pass keeps; the others' are finite."""
    from fovi_b200 import ops
    leaves, _ = _inputs(M, 96, 200, 80, dtype, M, bias=False)
    x, *weights = leaves[:4]
    weights = [w.abs() + 0.125 for w in weights]
    x[1, 5] = float("inf")
    for saved in (False, True):
        y, _ = ops.gated_feed_forward(x, *weights, activation=activation, want_saved=saved)
        assert (y[1] == float("inf")).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2:]).all()
