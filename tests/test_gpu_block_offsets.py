"""GPU: the operators of a token block where an offset in a tensor passes 2^31 values: rows far apart, and results and hidden values that are that large."""
import pytest
import torch

from oracle import block_oracle as oracle

pytestmark = pytest.mark.gpu
BF, F32, I8 = torch.bfloat16, torch.float32, torch.int8


@pytest.fixture(autouse=True)
def memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def _apart(rows, dtype):
    """A copy of rows with 2^30 values and more from one to the next (8 bits: 2^31), on 16-byte boundaries."""
    m, n = rows.shape
    step = (1 << (31 if dtype is I8 else 30)) + 64
    far = torch.empty((m - 1) * step + n, dtype=dtype, device="cuda").as_strided((m, n), (step, 1))
    return far.copy_(rows)


def _r(*s, dtype=BF, scale=1.0):
    return (torch.randn(*s, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("C", [256, 250, 9000])
def test_norm_of_rows_far_apart(C, dtype):
    from fovi_b200 import ops
    x, r, dy, d2 = (_r(3, C, dtype=dtype) for _ in range(4))
    w = torch.rand(C, device="cuda")
    for i in range(2):
        a, b = (_apart(x, dtype), r) if i == 0 else (x, _apart(r, dtype))
        want, got = ops.rms_norm(x, w, 1e-6, r, want_rstd=True), ops.rms_norm(a, w, 1e-6, b, want_rstd=True)
        for p, q in zip(want + ops.rms_norm_int8(x, w, 1e-6, r), got + ops.rms_norm_int8(a, w, 1e-6, b)):
            assert torch.equal(p, q)
        del a, b
    far = _apart(x, dtype)
    assert all(torch.equal(p, q) for p, q in zip(ops.quantize(x), ops.quantize(far)))
    del far
    want = ops.rms_norm_backward(want[1], dy, d2, w, want[2])
    for i in range(3):
        args = [_apart(t, dtype) if j == i else t for j, t in enumerate((got[1], dy, d2))]
        assert all(torch.equal(p, q) for p, q in zip(want, ops.rms_norm_backward(*args, w, got[2])))
        del args


@pytest.mark.parametrize("tokens", [3, 40])
def test_product_of_rows_far_apart(tokens):
    from fovi_b200 import ops
    q, w = (torch.randint(-128, 128, (n, 80), device="cuda", dtype=I8) for n in (tokens, 3))
    s, ws = torch.rand(tokens, device="cuda"), torch.rand(3, device="cuda")
    want = ops.linear_int8(q, s, w, ws)
    assert torch.equal(want, ops.linear_int8(q, s, _apart(w, I8), ws))
    if tokens == 3:
        assert torch.equal(want, ops.linear_int8(_apart(q, I8), s, w, ws))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_block_of_rows_far_apart(dtype):
    from fovi_b200 import ops
    M, C, F, O = 3, 64, 3, 3
    leaves, dy = [_r(M, C, dtype=dtype), _r(F, C, dtype=dtype), _r(F, C, dtype=dtype), _r(O, F, dtype=dtype)], _r(M, O, dtype=dtype)
    want = ops.gated_feed_forward(*leaves)[0], *ops.gated_feed_forward(*leaves, want_saved=True)
    grads = ops.gated_feed_forward_backward(*leaves, want[2], dy)
    for i in range(5):
        far = [_apart(t, dtype) if j == i else t for j, t in enumerate(leaves + [dy])]
        y, saved = ops.gated_feed_forward(*far[:4], want_saved=True)
        assert torch.equal(y, want[1]) and torch.equal(ops.gated_feed_forward(*far[:4])[0], want[0])
        assert all(torch.equal(p, q) for p, q in zip(grads, ops.gated_feed_forward_backward(*far[:4], saved, far[4])))
        del far


def test_norms_of_many_rows():
    """1.7 million rows of 1280: the last ones as by themselves."""
    from fovi_b200 import ops
    rows, C = 1_700_000, 1280
    x, dy = (torch.randn(rows, C, device="cuda", dtype=BF) for _ in range(2))
    w = torch.rand(C, device="cuda")
    last = slice(rows - 300, rows)
    q, s = ops.quantize(x)
    assert all(torch.equal(p[last], o) for p, o in zip((q, s), ops.quantize(x[last])))
    del q, s
    y, total, rstd = ops.rms_norm(x, w, residual=dy, want_rstd=True)
    assert all(torch.equal(p[last], o) for p, o in zip((y, total, rstd), ops.rms_norm(x[last], w, residual=dy[last], want_rstd=True)))
    dx, _ = ops.rms_norm_backward(total, dy, x, w, rstd)
    assert torch.equal(dx[last], ops.rms_norm_backward(total[last], dy[last], x[last], w, rstd[last])[0])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_product_of_many_rows(dtype):
    from fovi_b200 import ops
    M, K, N = 500_009, 32, 5120
    q, w = (torch.randint(-128, 128, (n, K), device="cuda", dtype=I8) for n in (M, N))
    s, ws = torch.rand(M, device="cuda"), torch.rand(N, device="cuda")
    y = ops.linear_int8(q, s, w, ws, None, dtype)
    assert torch.equal(y[-300:], ops.linear_int8(q[-300:], s[-300:], w, ws, None, dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_block_of_many_hidden_values(dtype):
    """1.1 million tokens of 2048 hidden values; only the last ones have a gradient, so that all gradients are theirs."""
    from fovi_b200 import ops
    M, C, F, O, last = 1_100_000, 32, 2048, 40, 300
    leaves = [_r(M, C, dtype=dtype), _r(F, C, dtype=dtype, scale=C ** -0.5), _r(F, C, dtype=dtype, scale=C ** -0.5), _r(O, F, dtype=dtype, scale=F ** -0.5)]
    dy = torch.zeros(M, O, device="cuda", dtype=dtype)
    dy[-last:] = _r(last, O, dtype=dtype)
    y, saved = ops.gated_feed_forward(*leaves, want_saved=True)
    dx, *grads = ops.gated_feed_forward_backward(*leaves, saved, dy)
    want = oracle.feed_forward(leaves[0][-last:], *leaves[1:], None, None, None, "silu", dy[-last:])
    for got, w in zip([y[-last:], dx[-last:]] + grads, want, strict=True):
        oracle.near(got, w)
    assert not dx[:-last].any()
    oracle.near(ops.gated_feed_forward(*leaves)[0][-last:], want[0])
