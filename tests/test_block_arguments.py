"""CPU: the entry points of a token block's operators refuse bad arguments before any CUDA call, and have no CPU path."""
import pytest
import torch

BAD, OK = 1, 0
P = 4096          # an address that nothing reads: every call below ends in front of its first launch


def _lib():
    from fovi_b200._lib import lib
    return lib


def _each(call, good, changes):
    for i, v in changes:
        args = list(good)
        args[i] = v
        assert call(*args) == BAD, (i, v)


def test_rms_norm():
    f = _lib().fovi_rms_norm_forward
    # x, dtype, rows, C, x_stride, residual, stride, weight, eps, total, y, q, q_stride, scale, rstd, stream
    good = [P, 1, 0, 8, 8, None, 0, None, 1e-6, None, P, None, 0, None, None, None]
    assert f(*good) == OK                                            # no rows: nothing to do
    _each(f, good, [(1, 2), (1, -1), (2, -1), (3, 0), (4, -1), (6, -1), (8, -1.0), (8, float("nan"))])
    good[2] = 4
    _each(f, good, [(0, None), (10, None), (11, P), (5, P), (9, P)])           # neither or both results, a residual without its sum and the other way round
    eight = good[:10] + [None, P, 8, P, None, None]
    _each(f, eight, [(12, 7), (13, None)])
    b = _lib().fovi_rms_norm_backward
    # t, dtype, rows, C, t_stride, dy, dy_stride, dt, dt_stride, weight, rstd, dx, dweight, work, work_bytes, stream
    good = [P, 0, 4, 8, 8, P, 8, None, 0, None, P, P, P, P, 1 << 20, None]
    _each(b, good, [(0, None), (1, 3), (2, -1), (3, 0), (4, -1), (5, None), (6, -1), (8, -1), (10, None), (13, None), (14, 4)])
    assert _lib().fovi_rms_norm_workspace_bytes(-1, 8) == -1 == _lib().fovi_rms_norm_workspace_bytes(4, 0)
    q = _lib().fovi_quantize_rows
    good = [P, 1, 4, 8, 8, P, 16, P, None]
    _each(q, good, [(0, None), (1, 2), (2, -1), (3, 0), (4, -1), (5, None), (6, 7), (7, None)])


def test_linear_int8():
    f = _lib().fovi_linear_int8
    # q, tokens, K, q_stride, scale, weight, N, weight_stride, weight_scale, bias, y, y_dtype, stream
    good = [P, 0, 32, 32, P, P, 8, 32, P, None, P, 1, None]
    assert f(*good) == OK
    _each(f, good, [(1, -1), (2, 0), (2, 131072), (3, -1), (6, 0), (7, -1), (11, 2)])
    good[1] = 4
    _each(f, good, [(0, None), (4, None), (5, None), (8, None), (10, None)])
    for i, v in ((0, P + 8), (3, 40), (5, P + 1), (7, 33), (10, P + 4)):
        args = list(good)
        args[i] = v
        assert f(*args) == 5


def test_gated_feed_forward():
    lib = _lib()
    f, b, size = lib.fovi_gated_ffn_forward, lib.fovi_gated_ffn_backward, lib.fovi_gated_ffn_workspace_bytes
    for dtype in (0, 1):
        assert f(P, dtype, 0, 8, 8, 8, 8, P, 8, P, 8, P, 8, None, None, None, 0, P, None, None, 0, None) == OK
    # x, dtype, tokens, C, F, O, x_stride, gate, stride, up, stride, down, stride, biases, activation, y, saved, work, bytes, stream
    good = [P, 1, 4, 16, 16, 16, 16, P, 16, P, 16, P, 16, None, None, None, 0, P, None, P, 1 << 20, None]
    _each(f, good, [(1, 2), (2, -1), (2, (1 << 30) + 1), (3, 0), (4, 0), (5, 0), (6, -1), (8, -1), (10, -1), (12, -1), (16, 2), (16, -1), (0, None), (7, None), (9, None), (11, None),
                    (17, None), (19, None), (20, 8)])
    # ... activation, saved, dy, dy_stride, dx, six more gradients, work, bytes, stream
    good = [P, 1, 4, 16, 16, 16, 16, P, 16, P, 16, P, 16, 0, P, P, 16, P, P, P, P, P, P, P, P, 1 << 30, None]
    _each(b, good, [(1, 2), (2, -1), (3, 0), (13, 2), (14, None), (15, None), (16, -1), (24, None), (25, 8), (0, None), (11, None)])
    for phase in (-1, 3, 7, 8):
        assert size(1, 4, 8, 8, 8, phase) == -1
    assert size(2, 4, 8, 8, 8, 0) == -1 == lib.fovi_gated_ffn_saved_bytes(1, -1, 8)
    for dtype in (0, 1):                                             # more rows never want less work, room for copies is room on top
        for phase in (0, 1, 2):
            assert size(dtype, 5, 40, 72, 24, phase) <= size(dtype, 500, 40, 72, 24, phase) <= size(dtype, 500, 40, 72, 24, phase + 4)


def test_no_cpu_path():
    from fovi_b200 import tokens
    x, w = torch.randn(4, 16), torch.randn(16, 16)
    q, s = torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)
    for call in (lambda: tokens.rms_norm(x), lambda: tokens.rms_norm_int8(x), lambda: tokens.quantize(x), lambda: tokens.linear_int8(q, s, q, s), lambda: tokens.gated_feed_forward(x, w, w, w)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="activation"):
        tokens.GatedFeedForward(8, 8, activation="relu", device="cpu")


def test_parts_of_a_float32_value():
    """csrc/product_split.cu cuts a value's 24 bits in three bf16 parts: they add up to the value, and what six of their nine products leave out is below a float32 product's rounding."""
    g = torch.Generator().manual_seed(1)
    x = torch.cat([torch.randn(20000, generator=g), torch.randn(1000, generator=g) * 1e30, torch.randn(1000, generator=g) * 1e-25,
                   torch.tensor([0.0, 1.0, 1.99999988, 1.00390625, 1.00390637, 3.4028234663852886e38, -3.4028234663852886e38])])

    def parts(v):
        out = []
        for _ in range(3):
            p = v.clamp(-torch.finfo(torch.bfloat16).max, torch.finfo(torch.bfloat16).max).to(torch.bfloat16).float()      # rounded without leaving the range
            out.append(p)
            v = v - p
        assert not v.any()
        return [p.double() for p in out]
    a, b = parts(x), parts(x.flip(0))
    for p in a:
        assert torch.isfinite(p).all() and torch.equal(p.to(torch.bfloat16).double(), p)
    assert torch.equal(sum(a), x.double())
    six = sum(a[i] * b[j] for i in range(3) for j in range(3) if i + j < 3)
    whole = x.double() * x.flip(0).double()
    far = (x.abs() > 3.39e38) | (x.flip(0).abs() > 3.39e38)                 # cut off where rounding would leave the range: a second part of up to 2^-7, a third of up to 2^-15 of the value
    # |second| <= 2^-8, |third| <= 2^-17 of the value: left out are two products of a second and a third part, and one of two third ones
    assert ((six - whole).abs() <= torch.where(far, 2.0 ** -21, 2.0 ** -24 + 2.0 ** -33) * whole.abs()).all()


def test_sizes_that_32_bits_do_not_count():
    """Refused before anything is read or launched: columns are counted in 32 bits, with a block's or a tile's width beyond the last one."""
    lib = _lib()
    for c in ((1 << 30) + 1, (1 << 31) - 1):
        for rows in (0, 1):
            assert lib.fovi_rms_norm_forward(P, 1, rows, c, c, None, 0, None, 1e-6, None, P, None, 0, None, None, None) == BAD
            assert lib.fovi_rms_norm_backward(P, 1, rows, c, c, P, c, None, 0, None, P, P, None, None, 0, None) == BAD
            assert lib.fovi_quantize_rows(P, 1, rows, c, c, P, c, P, None) == BAD
            assert lib.fovi_linear_int8(P, rows, 32, 32, P, P, c, 32, P, None, P, 1, None) == BAD
        assert lib.fovi_rms_norm_workspace_bytes(1, c) == -1
    for c in ((1 << 24) + 1, (1 << 31) - 1):
        for sizes in ((c, 8, 8), (8, c, 8), (8, 8, c)):
            for dtype in (0, 1):
                assert all(lib.fovi_gated_ffn_workspace_bytes(dtype, 1, *sizes, phase) == -1 for phase in (0, 1, 2))
                for tokens in (0, 1):
                    assert lib.fovi_gated_ffn_forward(P, dtype, tokens, *sizes, c, P, c, P, c, P, c, None, None, None, 0, P, None, P, 1 << 50, None) == BAD
                    assert lib.fovi_gated_ffn_backward(P, dtype, tokens, *sizes, c, P, c, P, c, P, c, 0, P, P, c, P, P, P, P, P, P, P, P, 1 << 50, None) == BAD
        assert lib.fovi_gated_ffn_saved_bytes(1, 1, c) == -1


def test_sizes_that_python_refuses(monkeypatch):
    from fovi_b200 import ops
    monkeypatch.setattr(ops, "_need_cuda", lambda *a: None)
    BF, F32, I8 = torch.bfloat16, torch.float32, torch.int8

    def t(dtype, *s): return torch.empty(*s, dtype=dtype, device="meta")
    n = (1 << 30) + 1
    for call in (lambda: ops.rms_norm(t(BF, 1, n)), lambda: ops.quantize(t(BF, 1, n)), lambda: ops.linear_int8(t(I8, 4, 16), t(F32, 4), t(I8, n, 16), t(F32, n)),
                 lambda: ops.linear_int8(t(I8, n, 16), t(F32, n), t(I8, 4, 16), t(F32, 4))):
        with pytest.raises(ValueError, match="2.30"):
            call()
    n = (1 << 24) + 1
    for c, h, o in ((n, 8, 8), (8, n, 8), (8, 8, n)):
        with pytest.raises(ValueError, match="2.24"):
            ops.gated_feed_forward(t(BF, 1, c), t(BF, h, c), t(BF, h, c), t(BF, o, h))
