"""GPU: layer norm over the last axis and its gradients against the definition in 64 bits."""
import pytest
import torch

from oracle import token_oracle as oracle

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True, params=["native", "python"])
def launch_path(request, monkeypatch):
    """Every test with the native launch path (csrc/bind_tokens.h) and with the Python one."""
    from fovi_b200 import ops
    assert ops._native is not None
    if request.param == "python":
        monkeypatch.setattr(ops, "_native", None)


def _inputs(rows, C, dtype, seed, offset=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, C, generator=g, device="cuda") + offset).to(dtype)
    w = torch.rand(C, generator=g, device="cuda") + 0.5
    b = torch.randn(C, generator=g, device="cuda")
    return x, w, b, torch.randn(rows, C, generator=g, device="cuda").to(dtype)


SIZES = [(1, 1), (1, 384), (7, 2), (65, 384), (33, 1280), (130, 768), (5, 1000), (19, 1023), (3, 4096), (2, 8200), (1031, 96), (700, 31), (4100, 8), (2500, 384),
         (1300, 1280), (600, 2048), (300, 4104)]


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,C", SIZES)
def test_forward_and_gradients(rows, C, dtype):
    from fovi_b200 import tokens
    x, w, b, dy = _inputs(rows, C, dtype, rows + C)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = tokens.layer_norm(*leaves, eps=1e-6)
    assert y.dtype is dtype and y.is_contiguous()
    got = (y,) + torch.autograd.grad(y, leaves, dy)
    for g, want in zip(got, oracle.layer_norm(x.detach(), w.detach(), b.detach(), 1e-6, dy)):
        oracle.near(g.detach(), want)
    with torch.no_grad():
        assert torch.equal(tokens.layer_norm(x, w, b, eps=1e-6), y)


@pytest.mark.autograd
@pytest.mark.parametrize("C", [64, 100, 384, 1280, 5000])
@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_without_parameters(C, which):
    from fovi_b200 import tokens
    x, w, b, dy = _inputs(37, C, F32, C)
    w, b = (w if which == "weight" else None), (b if which == "bias" else None)
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = tokens.layer_norm(x, w, b)
    got = torch.autograd.grad(y, leaves, dy)
    want = oracle.layer_norm(x.detach(), w, b, 1e-5, dy)
    oracle.near(y.detach(), want[0])
    oracle.near(got[0], want[1])
    if len(got) > 1:
        oracle.near(got[1], want[2 if which == "weight" else 3])


@pytest.mark.parametrize("x_dtype,y_dtype", [(F32, BF), (BF, F32)])
@pytest.mark.parametrize("C", [384, 100, 3000])
def test_result_of_another_type(x_dtype, y_dtype, C):
    from fovi_b200 import ops
    x, w, b, dy = _inputs(50, C, x_dtype, 3)
    dy = dy.to(y_dtype)
    y, stats = ops.layer_norm(x, w, b, 1e-6, y_dtype, want_stats=True)
    assert y.dtype is y_dtype
    got = (y,) + ops.layer_norm_backward(x, dy, w, stats)
    assert got[1].dtype is x_dtype
    for g, want in zip(got, oracle.layer_norm(x, w, b, 1e-6, dy, y_dtype)):
        oracle.near(g, want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strided_rows(dtype):
    """Slices whose rows are further apart than they are long, aligned and not; an expanded gradient; a column slice."""
    from fovi_b200 import ops
    x, w, b, dy = _inputs(40, 400, dtype, 5)
    for lo, hi in ((0, 384), (8, 392), (1, 385), (3, 100)):
        xs, gs, ws, bs = x[:, lo:hi], dy[:, lo:hi], w[lo:hi], b[lo:hi]
        y, stats = ops.layer_norm(xs, ws, bs, 1e-6, want_stats=True)
        for g, want in zip((y,) + ops.layer_norm_backward(xs, gs, ws, stats), oracle.layer_norm(xs, ws, bs, 1e-6, gs)):
            oracle.near(g, want)
    same = dy[:1].expand(40, 400)
    y, stats = ops.layer_norm(x, w, b, 1e-6, want_stats=True)
    for g, want in zip((y,) + ops.layer_norm_backward(x, same, w, stats), oracle.layer_norm(x, w, b, 1e-6, same)):
        oracle.near(g, want)
    xt, gt = x.t(), dy.t()
    y, stats = ops.layer_norm(xt, None, None, 1e-6, want_stats=True)
    for g, want in zip((y,) + ops.layer_norm_backward(xt, gt, None, stats), oracle.layer_norm(xt, None, None, 1e-6, gt)):
        oracle.near(g, want)


def test_a_large_common_offset_costs_no_digits():
    """Values around 4096 with a spread of one: the variance is taken about the mean."""
    from fovi_b200 import tokens
    x, w, b, _ = _inputs(20, 384, F32, 6, offset=4096.0)
    oracle.near(tokens.layer_norm(x, w, b), oracle.layer_norm(x, w, b, 1e-5))


def test_equal_values_and_not_a_number():
    from fovi_b200 import tokens
    x = torch.full((3, 384), 2.5, device="cuda")
    x[1, 7] = float("nan")
    x[2] = 0
    y = tokens.layer_norm(x)
    assert torch.equal(y[0], torch.zeros_like(y[0])) and torch.isnan(y[1]).all() and torch.equal(y[2], torch.zeros_like(y[2]))


@pytest.mark.autograd
def test_no_rows_and_many_axes():
    from fovi_b200 import tokens
    x, w, b, _ = _inputs(0, 16, F32, 1)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = tokens.layer_norm(*leaves)
    gx, gw, gb = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert y.shape == (0, 16) and gx.shape == (0, 16) and not gw.any() and not gb.any()
    x = torch.randn(2, 3, 5, 24, device="cuda")
    with torch.no_grad():
        assert torch.equal(tokens.layer_norm(x, w[:8].repeat(3), b[:8].repeat(3)),
                           tokens.layer_norm(x.view(30, 24), w[:8].repeat(3), b[:8].repeat(3)).view(x.shape))


def test_parameter_gradients_are_the_same_bits():
    from fovi_b200 import ops
    for rows, C in ((5000, 384), (3000, 1280), (900, 100)):
        x, w, b, dy = _inputs(rows, C, BF, 9)
        _, stats = ops.layer_norm(x, w, b, want_stats=True)
        first = ops.layer_norm_backward(x, dy, w, stats)
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(first, ops.layer_norm_backward(x, dy, w, stats)))


@pytest.mark.autograd
def test_module_on_another_stream_and_bf16_parameters():
    from fovi_b200.tokens import TokenNorm
    stream = torch.cuda.Stream()
    m = TokenNorm(384, dtype=BF)
    m.load_state_dict({"weight": torch.rand(384) + 0.5, "bias": torch.randn(384)})
    x, _, _, dy = _inputs(77, 384, BF, 12)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = m(x.requires_grad_(True))
        y.backward(dy)
    torch.cuda.current_stream().wait_stream(stream)
    want = oracle.layer_norm(x.detach(), m.weight.detach(), m.bias.detach(), 1e-6, dy)
    oracle.near(y.detach(), want[0])
    oracle.near(x.grad, want[1])
    assert m.weight.grad.dtype is BF and m.bias.grad.dtype is BF
    for got, (value, bound) in ((m.weight.grad, want[2]), (m.bias.grad, want[3])):      # rounded once more, to the parameter's type
        oracle.near(got, (value, bound + oracle.U16 * (value.abs() + bound)))


def test_gradient_against_differences():
    """Central differences of the kernel's own forward pass along a random direction; the difference between two step sizes bounds the truncation."""
    from fovi_b200 import ops
    x, w, b, dy = _inputs(9, 48, F32, 21)
    g = torch.Generator(device="cuda").manual_seed(1)
    dirs = [torch.randn(t.shape, generator=g, device="cuda") for t in (x, w, b)]
    _, stats = ops.layer_norm(x, w, b, want_stats=True)
    grads = ops.layer_norm_backward(x, dy, w, stats)
    for i in range(3):
        def loss(h):
            args = [t + h * d if j == i else t for j, (t, d) in enumerate(zip((x, w, b), dirs))]
            return (ops.layer_norm(*args).double() * dy.double()).sum().item()
        near, far = ((loss(h) - loss(-h)) / (2 * h) for h in (2.0 ** -7, 2.0 ** -6))
        rounding = 32 * oracle.U32 * dy.double().abs().sum().item() * 4 / 2.0 ** -7
        assert abs((grads[i].double() * dirs[i].double()).sum().item() - near) <= abs(near - far) + rounding


def test_refusals():
    from fovi_b200 import ops, tokens
    x = torch.randn(4, 16, device="cuda")
    with pytest.raises(ValueError, match="CUDA"):
        tokens.layer_norm(x.cpu())
    with pytest.raises(ValueError, match="CUDA"):
        tokens.layer_norm(x, torch.ones(16))
    with pytest.raises(ValueError, match="weight has 8"):
        tokens.layer_norm(x, torch.ones(8, device="cuda"))
    with pytest.raises(ValueError, match="eps"):
        tokens.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        tokens.layer_norm(x, eps=float("nan"))
    with pytest.raises(ValueError, match="last axis"):
        tokens.layer_norm(x[:, :0])
    with pytest.raises(TypeError, match="dtype"):
        tokens.layer_norm(x.half())
    with pytest.raises(ValueError, match="shape"):
        ops.layer_norm_backward(x, x[:, :8], None, torch.zeros(4, 2, device="cuda"))
    with pytest.raises(ValueError, match="stats"):
        ops.layer_norm_backward(x, x, None, torch.zeros(3, 2, device="cuda"))
