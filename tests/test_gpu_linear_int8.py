"""GPU: the product of 8-bit tokens with 8-bit weights against the definition in 64 bits."""
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


def _inputs(m, k, n, seed, low=-128):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, w = (torch.randint(low, 128, (r, k), generator=g, device="cuda", dtype=torch.int8) for r in (m, n))
    s, ws = (torch.rand(r, generator=g, device="cuda") + 0.1 for r in (m, n))
    return q, s, w, ws, torch.randn(n, generator=g, device="cuda") * 50


SIZES = [(1, 1, 1), (1, 16, 8), (1, 1280, 5120), (2, 384, 384), (5, 100, 33), (8, 1280, 1280), (9, 131, 64), (16, 48, 250), (17, 384, 1000), (31, 1003, 77), (33, 16, 16), (64, 4112, 96),
         (65, 384, 384), (100, 37, 513), (128, 128, 256), (129, 1280, 384), (257, 640, 130), (300, 2000, 1031), (1031, 1003, 331), (2600, 384, 96), (777, 5120, 640), (48, 1280, 1280), (200, 96, 250), (1000, 64, 40), (1030, 48, 24)]


@pytest.mark.parametrize("out_dtype", [BF, F32])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_product(m, k, n, out_dtype):
    from fovi_b200 import tokens
    q, s, w, ws, b = _inputs(m, k, n, m + k + n)
    for bias in (None, b):
        y = tokens.linear_int8(q, s, w, ws, bias, out_dtype=out_dtype)
        assert y.dtype is out_dtype and y.is_contiguous()
        oracle.near(y, oracle.linear_int8(q, s, w, ws, bias, out_dtype))


@pytest.mark.parametrize("m", [1, 40, 700])
def test_largest_values(m):
    """Sums at the end of what 32 bits hold: -128 times -128, 131071 times."""
    from fovi_b200 import tokens
    k, n = 131071, 20
    q, w = torch.full((m, k), -128, dtype=torch.int8, device="cuda"), torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    w[1] = 127
    one_m, one_n = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    y = tokens.linear_int8(q, one_m, w, one_n, out_dtype=F32)
    want = torch.full((m, n), float(128 * 128 * k), device="cuda")
    want[:, 1] = float(-128 * 127 * k)
    assert torch.equal(y, want)


@pytest.mark.parametrize("m", [3, 200])
def test_strides_and_shapes(m):
    from fovi_b200 import tokens
    q, s, w, ws, b = _inputs(m, 420, 90, m)
    for lo, hi in ((0, 400), (16, 416), (1, 385), (3, 100)):
        oracle.near(tokens.linear_int8(q[:, lo:hi], s, w[:, lo:hi], ws, b), oracle.linear_int8(q[:, lo:hi], s, w[:, lo:hi], ws, b, BF))
    want = oracle.linear_int8(q, s, w, ws, b, BF)
    oracle.near(tokens.linear_int8(q.t().contiguous().t(), s, w.t().contiguous().t(), ws, b), want)
    oracle.near(tokens.linear_int8(q, torch.stack([s, s], 1)[:, 0], w, torch.stack([ws, ws], 1)[:, 1], b.to(BF).float()), oracle.linear_int8(q, s, w, ws, b.to(BF), BF))
    same = q[:1].expand(m, 420)
    oracle.near(tokens.linear_int8(same, s, w, ws), oracle.linear_int8(same, s, w, ws, None, BF))
    same = w[:1].expand(90, 420)
    oracle.near(tokens.linear_int8(q, s, same, ws), oracle.linear_int8(q, s, same, ws, None, BF))
    whole = tokens.linear_int8(q, s, w, ws, b)
    assert torch.equal(tokens.linear_int8(q[:, None, None], s[:, None, None], w, ws, b), whole[:, None, None])
    assert torch.equal(tokens.linear_int8(q[0], s[0], w, ws, b), tokens.linear_int8(q[:1], s[:1], w, ws, b)[0])
    assert tokens.linear_int8(q[:0], s[:0], w, ws, b).shape == (0, 90)


def test_a_row_whose_scale_is_no_number():
    from fovi_b200 import tokens
    for m in (2, 300):
        q, s, w, ws, b = _inputs(m, 64, 48, 3)
        want = tokens.linear_int8(q, s, w, ws, b)
        s[1] = float("nan")
        y = tokens.linear_int8(q, s, w, ws, b)
        assert torch.isnan(y[1]).all() and torch.equal(y[0], want[0]) and torch.equal(y[2:], want[2:])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m", [1, 65, 300])
def test_layer(m, dtype):
    """Linear8 made from a linear layer: of tensors, and of what the norm gives in 8 bits; cast with its model its scales stay what they are."""
    from fovi_b200 import tokens
    torch.manual_seed(m)
    linear = torch.nn.Linear(200, 72, device="cuda")
    layer = tokens.Linear8(linear, out_dtype=dtype)
    x, res = (torch.randn(m, 200, device="cuda").to(dtype) for _ in range(2))
    wq, ws = tokens.quantize(linear.weight)
    q, s = tokens.quantize(x)
    want = oracle.linear_int8(q, s, wq, ws, linear.bias, dtype)
    oracle.near(layer(x), want)
    assert torch.equal(layer(q, s), layer(x))
    q, s, _ = tokens.rms_norm_int8(x, residual=res)
    oracle.near(layer(q, s), oracle.linear_int8(q, s, wq, ws, linear.bias, dtype))
    y = layer(x)
    again = tokens.Linear8(torch.nn.Linear(200, 72, device="cuda"), out_dtype=dtype)
    again.load_state_dict(layer.state_dict())
    assert torch.equal(again(x), y)
    assert layer.to(BF).weight_scale.dtype is F32 and layer.bias.dtype is F32 and torch.equal(layer(x), y)
    # against the layer itself: half a step on each side, in every product
    value = x.double() @ linear.weight.double().T + linear.bias.double()
    qs, sd = tokens.quantize(x)[1].double()[:, None], ws.double()
    e = 0.51 * (qs * linear.weight.double().abs().sum(1) + sd * x.double().abs().sum(1, keepdim=True) + 200 * qs * sd)
    oracle.near(y, (value, e + 2 * oracle.U16 * (value.abs() + e)))


@pytest.mark.autograd
def test_refusals():
    from fovi_b200 import tokens
    q, s, w, ws, b = _inputs(4, 32, 8, 1)
    ok = dict(q=q, scale=s, weight=w, weight_scale=ws, bias=b)
    bad = [(ValueError, "CUDA", dict(q=q.cpu())), (ValueError, "CUDA", dict(weight=w.cpu())), (ValueError, "CUDA", dict(scale=s.cpu())), (ValueError, "CUDA", dict(bias=b.cpu())),
           (TypeError, "int8", dict(q=q.to(torch.uint8))), (TypeError, "int8", dict(weight=w.float())), (TypeError, "float32", dict(scale=s.double())),
           (TypeError, "float32", dict(weight_scale=ws.bfloat16())), (ValueError, "wanted", dict(weight=w[:, :16])), (ValueError, "wanted", dict(weight=w[0])),
           (ValueError, "wanted", dict(weight=w[:0], weight_scale=ws[:0])), (ValueError, "wanted", dict(q=q[:, :0], weight=w[:, :0])),
           (ValueError, "one for each", dict(scale=s[:1])), (ValueError, "one for each", dict(weight_scale=ws[:1])), (ValueError, "one for each", dict(scale=s[:, None])),
           (ValueError, "bias has 4", dict(bias=b[:4])), (TypeError, "dtype", dict(out_dtype=torch.float16)),
           (NotImplementedError, "no gradient", dict(scale=s.clone().requires_grad_(True))), (NotImplementedError, "no gradient", dict(bias=b.clone().requires_grad_(True)))]
    for error, words, change in bad:
        with pytest.raises(error, match=words):
            tokens.linear_int8(**{**ok, **change})
    long = torch.zeros(1, 131072, dtype=torch.int8, device="cuda")
    with pytest.raises(ValueError, match="131071"):
        tokens.linear_int8(long, s[:1], long, ws[:1])
