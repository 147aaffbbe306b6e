"""GPU: root-mean-square norm with the residual's addition, its gradients and its 8-bit form, against the definition in 64 bits."""
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


def _inputs(rows, C, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    def n(*s): return torch.randn(*s, generator=g, device="cuda")
    x, res, dy, dt = ((n(rows, C) + o).to(dtype) for o in (0.0, 0.5, 0.0, 0.0))
    return x, res, torch.rand(C, generator=g, device="cuda") + 0.5, dy, dt


SIZES = [(1, 1), (1, 384), (7, 2), (65, 384), (33, 1280), (130, 768), (5, 1000), (19, 1023), (3, 4096), (2, 8200), (1031, 96), (700, 31), (4100, 8), (2500, 384),
         (1300, 1280), (600, 2048), (300, 4104), (9, 520), (40, 516)]


@pytest.mark.autograd
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,C", SIZES)
def test_forward_and_gradients(rows, C, dtype, residual):
    from fovi_b200 import tokens
    x, res, w, dy, dt = _inputs(rows, C, dtype, rows + C)
    res, dt = (res, dt) if residual else (None, None)
    leaves = [t.requires_grad_(True) for t in (x, w, res) if t is not None]
    outs = tokens.rms_norm(x, w, eps=1e-6, residual=res)
    outs = outs if residual else (outs,)
    assert all(o.dtype is dtype and o.is_contiguous() and o.shape == x.shape for o in outs)
    grads = torch.autograd.grad(outs, leaves, (dy, dt) if residual else (dy,))
    got = outs + grads[:2]
    for g, want in zip(got, oracle.rms_norm(x.detach(), w.detach(), 1e-6, None if res is None else res.detach(), dy, dt), strict=True):
        oracle.near(g.detach(), want)
    if residual:
        assert torch.equal(grads[0], grads[2])
    with torch.no_grad():
        again = tokens.rms_norm(x, w, eps=1e-6, residual=res)
        assert all(torch.equal(p, q) for p, q in zip(again if residual else (again,), outs))
        if residual:                                 # the two calls, one after the other
            assert torch.equal(outs[1], x + res) and torch.equal(outs[0], tokens.rms_norm(x + res, w, eps=1e-6))


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,C", SIZES)
def test_eight_bits(rows, C, dtype, residual):
    from fovi_b200 import tokens
    x, res, w, _, _ = _inputs(rows, C, dtype, rows + C + 1)
    res = res if residual else None
    q, scale, *total = tokens.rms_norm_int8(x, w, residual=res)
    want = oracle.rms_norm(x, w, 1e-6, res)
    y = want[0][0]
    oracle.near_eight_bits(q, scale, y, y.abs() * (C + 20) * oracle.U32)
    assert len(total) == residual and all(torch.equal(t, x + res) for t in total)
    assert q.data_ptr() % 16 == 0 and (q.stride(0) % 16 == 0 or rows == 1)
    q, scale = tokens.quantize(x)
    oracle.near_eight_bits(q, scale, x.double(), torch.zeros_like(x, dtype=torch.float64))


@pytest.mark.autograd
@pytest.mark.parametrize("C", [64, 100, 384, 1280, 9000])
def test_which_gradients_are_asked_for(C):
    """Without a weight; the norm's or the sum's result alone; one of the inputs alone."""
    from fovi_b200 import tokens
    x, res, w, dy, dt = _inputs(37, C, F32, C)
    for t in (x, res, w):
        t.requires_grad_(True)
    y, total = tokens.rms_norm(x, None, residual=res)
    dx, = torch.autograd.grad((y, total), (x,), (dy, dt))
    oracle.near(dx, oracle.rms_norm(x.detach(), None, 1e-6, res.detach(), dy, dt)[2])
    y, total = tokens.rms_norm(x, w, residual=res)
    want = oracle.rms_norm(x.detach(), w.detach(), 1e-6, res.detach(), dy, None)
    dr, dw = torch.autograd.grad(y, (res, w), dy, retain_graph=True)
    oracle.near(dr, want[2])
    oracle.near(dw, want[3])
    got = torch.autograd.grad(total, (x, res, w), dt, retain_graph=True, allow_unused=True)
    assert torch.equal(got[0], dt) and torch.equal(got[1], dt) and (got[2] is None or not got[2].any())
    assert torch.equal(torch.autograd.grad(y, w, dy)[0], dw)
    y = tokens.rms_norm(x, w)
    assert torch.equal(torch.autograd.grad(y, w, dy, retain_graph=True)[0], torch.autograd.grad(y, (x, w), dy)[1])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strided_rows(dtype):
    """Slices whose rows are further apart than they are long, aligned and not; expanded tensors; a column slice."""
    from fovi_b200 import ops
    x, res, w, dy, dt = _inputs(40, 400, dtype, 5)

    def both(xs, rs, ws, gs, ts):
        y, total, rstd = ops.rms_norm(xs, ws, 1e-6, rs, want_rstd=True)
        got = (y, total) + ops.rms_norm_backward(total, gs, ts, ws, rstd)
        for g, want in zip(got, oracle.rms_norm(xs, ws, 1e-6, rs, gs, ts), strict=True):
            oracle.near(g, want)
        q, scale, total8 = ops.rms_norm_int8(xs, ws, 1e-6, rs)
        value = oracle.rms_norm(xs, ws, 1e-6, rs)[0][0]
        oracle.near_eight_bits(q, scale, value, value.abs() * (xs.shape[1] + 20) * oracle.U32)
        assert torch.equal(total8, total)
    for lo, hi in ((0, 384), (8, 392), (1, 385), (3, 100)):
        both(x[:, lo:hi], res[:, lo:hi], w[lo:hi], dy[:, lo:hi], dt[:, lo:hi])
        both(x[:, lo:hi], res[:, :hi - lo], w[lo:hi], dy[:, lo:hi].contiguous(), dt[:, 400 - hi + lo:])
    both(x, res[:1].expand(40, 400), w, dy[:1].expand(40, 400), dt[:1].expand(40, 400))
    both(x.t(), res.t(), None, dy.t(), dt.t())


def test_zeros_and_values_that_are_no_numbers():
    from fovi_b200 import tokens
    for C in (384, 100, 9000):
        x = torch.ones(5, C, device="cuda")
        x[0], x[1, 7], x[2, 3], x[3] = 0, float("nan"), float("inf"), 1e-42
        y = tokens.rms_norm(x)
        assert not y[0].any() and torch.isnan(y[1]).all() and torch.isnan(y[2, 3]) and torch.isfinite(y[3:]).all()
        for q, scale in (tokens.rms_norm_int8(x), tokens.quantize(x)):
            assert not q[0].any() and scale[0] == torch.finfo(F32).tiny
            assert not torch.isfinite(scale[1:3]).any() and torch.isfinite(scale[3:]).all() and (q[4] == 127).all()


@pytest.mark.autograd
def test_no_rows_and_many_axes():
    from fovi_b200 import tokens
    x, res, w, _, _ = _inputs(0, 16, F32, 1)
    leaves = [t.requires_grad_(True) for t in (x, res, w)]
    y, total = tokens.rms_norm(x, w, residual=res)
    gx, gr, gw = torch.autograd.grad((y, total), leaves, (torch.ones_like(y), torch.ones_like(y)))
    assert y.shape == total.shape == gx.shape == gr.shape == (0, 16) and not gw.any()
    with torch.no_grad():
        q, scale = tokens.rms_norm_int8(x, w)
        assert q.shape == (0, 16) and scale.shape == (0,)
        x = torch.randn(2, 3, 5, 24, device="cuda")
        w = torch.rand(24, device="cuda")
        assert torch.equal(tokens.rms_norm(x, w), tokens.rms_norm(x.view(30, 24), w).view(x.shape))
        q, scale = tokens.rms_norm_int8(x, w)
        assert q.shape == x.shape and scale.shape == x.shape[:-1]
        assert tokens.quantize(x[0, 0, 0])[1].shape == ()


def test_gradients_are_the_same_bits():
    from fovi_b200 import ops
    for rows, C in ((5000, 384), (3000, 1280), (900, 100)):
        x, res, w, dy, dt = _inputs(rows, C, BF, 9)
        _, total, rstd = ops.rms_norm(x, w, 1e-6, res, want_rstd=True)
        first = ops.rms_norm_backward(total, dy, dt, w, rstd)
        for _ in range(3):
            assert all(torch.equal(p, q) for p, q in zip(first, ops.rms_norm_backward(total, dy, dt, w, rstd)))


def test_gradient_against_differences():
    """Central differences of the kernel's own forward pass along a random direction; the difference between two step sizes bounds the truncation."""
    from fovi_b200 import ops
    x, _, w, dy, _ = _inputs(9, 48, F32, 21)
    g = torch.Generator(device="cuda").manual_seed(1)
    dirs = [torch.randn(t.shape, generator=g, device="cuda") for t in (x, w)]
    _, _, rstd = ops.rms_norm(x, w, want_rstd=True)
    grads = ops.rms_norm_backward(x, dy, None, w, rstd)
    for i in range(2):
        def loss(h):
            args = [t + h * d if j == i else t for j, (t, d) in enumerate(zip((x, w), dirs))]
            return (ops.rms_norm(*args)[0].double() * dy.double()).sum().item()
        near, far = ((loss(h) - loss(-h)) / (2 * h) for h in (2.0 ** -7, 2.0 ** -6))
        rounding = 32 * oracle.U32 * dy.double().abs().sum().item() * 4 / 2.0 ** -7
        assert abs((grads[i].double() * dirs[i].double()).sum().item() - near) <= abs(near - far) + rounding


@pytest.mark.autograd
def test_module_on_another_stream_and_bf16_parameters():
    from fovi_b200.tokens import TokenRMSNorm
    stream = torch.cuda.Stream()
    m = TokenRMSNorm(384, dtype=BF)
    m.load_state_dict(torch.nn.RMSNorm(384).state_dict())
    x, res, _, dy, dt = _inputs(77, 384, BF, 12)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y, total = m(x.requires_grad_(True), res.requires_grad_(True))
        torch.autograd.backward((y, total), (dy, dt))
    torch.cuda.current_stream().wait_stream(stream)
    want = oracle.rms_norm(x.detach(), m.weight.detach(), 1e-6, res.detach(), dy, dt)
    for got, w in zip((y, total, x.grad), want):
        oracle.near(got.detach(), w)
    assert torch.equal(x.grad, res.grad) and m.weight.grad.dtype is BF
    value, bound = want[3]                                                                  # rounded once more, to the parameter's type
    oracle.near(m.weight.grad, (value, bound + oracle.U16 * (value.abs() + bound)))


@pytest.mark.autograd
def test_refusals():
    from fovi_b200 import ops, tokens
    x = torch.randn(4, 16, device="cuda")
    for call in (tokens.rms_norm, tokens.rms_norm_int8):
        with pytest.raises(ValueError, match="CUDA"):
            call(x.cpu())
        with pytest.raises(ValueError, match="CUDA"):
            call(x, torch.ones(16))
        with pytest.raises(ValueError, match="CUDA"):
            call(x, residual=x.cpu())
        with pytest.raises(ValueError, match="weight has 8"):
            call(x, torch.ones(8, device="cuda"))
        with pytest.raises(ValueError, match="eps"):
            call(x, eps=-1.0)
        with pytest.raises(ValueError, match="last axis"):
            call(x[:, :0])
        with pytest.raises(TypeError, match="dtype"):
            call(x.half())
        with pytest.raises(ValueError, match="residual"):
            call(x, residual=x[:1])
        with pytest.raises(ValueError, match="residual"):
            call(x, residual=x.bfloat16())
    with pytest.raises(TypeError, match="dtype"):
        tokens.quantize(x.half())
    with pytest.raises(ValueError, match="CUDA"):
        tokens.quantize(x.cpu())
    with pytest.raises(ValueError, match="last axis"):
        tokens.quantize(x[:, :0])
    with pytest.raises(NotImplementedError, match="no gradient"):
        tokens.rms_norm_int8(x, torch.ones(16, device="cuda", requires_grad=True))
    with pytest.raises(NotImplementedError, match="no gradient"):
        tokens.quantize(x.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="shape"):
        ops.rms_norm_backward(x, x[:, :8], None, None, torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError, match="rstd"):
        ops.rms_norm_backward(x, x, None, None, torch.zeros(3, device="cuda"))
