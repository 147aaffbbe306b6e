"""GPU: rotary positions with several axes, and their gradient, against the definition in 64 bits."""
import math

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


def _inputs(B, L, H, D, pairs, prefix, shared, dtype, seed, reach=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, L, H, D, generator=g, device="cuda").to(dtype)
    n = L - prefix
    pos = (torch.rand((n, len(pairs)) if shared else (B, n, len(pairs)), generator=g, device="cuda") * 2 - 1) * reach
    f = 2 * math.pi * 100.0 ** (-torch.rand(sum(pairs), generator=g, device="cuda"))
    return x, pos, f


CASES = [  # B, L, H, D, pairs, prefix, shared
    (1, 1, 1, 2, (1,), 0, True), (2, 65, 6, 64, (16, 16), 1, False), (3, 17, 20, 64, (11, 11, 10), 5, True), (1, 1, 20, 64, (11, 11, 10), 0, False),
    (2, 33, 3, 80, (20, 20), 1, True), (2, 9, 2, 128, (10, 22, 32), 0, False), (1, 70, 5, 32, (4, 4, 4, 4), 2, True), (2, 7, 3, 48, (9, 8), 0, False),
    (2, 6, 2, 7, (1, 2), 0, True), (1, 5, 4, 96, (0, 16, 0), 1, False), (4, 3, 2, 64, (0,), 0, True), (2, 4, 2, 64, (16, 16), 4, True), (5, 130, 12, 64, (32,), 0, False),
    (1, 300, 1, 256, (64, 64), 3, False), (2, 40, 33, 16, (4, 4), 0, True)]


@pytest.mark.autograd
@pytest.mark.parametrize("pairing", ["halves", "pairs"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradient(case, dtype, pairing):
    from fovi_b200 import tokens
    B, L, H, D, pairs, prefix, shared = case
    x, pos, f = _inputs(*case, dtype, L + D)
    dy = torch.randn_like(x)
    x.requires_grad_(True)
    y = tokens.rotary(x, pos, f, pairs, prefix, pairing)
    gx, = torch.autograd.grad(y, x, dy)
    assert y.dtype is dtype and y.is_contiguous()
    inter = pairing == "pairs"
    oracle.near(y.detach(), oracle.rotary(x.detach(), pos, f, pairs, prefix, inter))
    oracle.near(gx, oracle.rotary(dy, pos, f, pairs, prefix, inter, inverse=True))
    assert torch.equal(y[:, :prefix], x[:, :prefix]) and torch.equal(y[..., 2 * sum(pairs):], x[..., 2 * sum(pairs):])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("pairing", ["halves", "pairs"])
def test_strides(dtype, pairing):
    """Heads in front of tokens, a slice of a packed projection, channels that are not contiguous, a start on no 16-byte boundary, an expanded batch, positions with strides."""
    from fovi_b200 import tokens
    inter = pairing == "pairs"
    x, pos, f = _inputs(2, 21, 6, 64, (16, 16), 1, False, dtype, 3)
    packed = torch.randn(2, 21, 3, 6, 64, device="cuda").to(dtype)
    odd = torch.randn(2, 21, 6, 65, device="cuda").to(dtype)[..., 1:]
    views = [x.transpose(1, 2).contiguous().transpose(1, 2), packed[:, :, 1], odd, x.transpose(2, 3).contiguous().transpose(2, 3), x[:1].expand(2, -1, -1, -1), x[:, :, ::2]]
    for v in views:
        oracle.near(tokens.rotary(v, pos, f, (16, 16), 1, pairing), oracle.rotary(v, pos, f, (16, 16), 1, inter))
    for p in (pos[:1].expand(2, -1, -1), torch.randn(2, 20, 4, device="cuda")[..., ::2], torch.randn(20, 2, 2, device="cuda").transpose(0, 1),
              torch.randn(2, 20, device="cuda").t()):
        oracle.near(tokens.rotary(x, p, f, (16, 16), 1, pairing), oracle.rotary(x, p, f, (16, 16), 1, inter))
    p = torch.randn(2, 40, 2, device="cuda")[:, ::2]
    oracle.near(tokens.rotary(x, p, f, (16, 16), 1, pairing), oracle.rotary(x, p, f, (16, 16), 1, inter))


def test_places_far_out():
    """Angles of some thousand turns keep float32's accuracy: the product's rounding error is carried."""
    from fovi_b200 import tokens
    x, pos, f = _inputs(1, 200, 2, 64, (16, 16), 0, True, F32, 8, reach=5000.0)
    oracle.near(tokens.rotary(x, pos, f, (16, 16)), oracle.rotary(x, pos, f, (16, 16)))


def test_turning_there_and_back_and_not_a_number():
    from fovi_b200 import ops
    x, pos, f = _inputs(2, 10, 4, 64, (16, 16), 0, True, F32, 4)
    back = ops.rotary(ops.rotary(x, pos, f, (16, 16)), pos, f, (16, 16), inverse=True)
    assert (back - x).abs().max() <= 32 * oracle.U32 * x.abs().max()
    x[1, 3, 2, 5] = float("nan")
    y = ops.rotary(x, pos, f, (16, 16))
    hit = torch.isnan(y).nonzero().tolist()
    assert hit == [[1, 3, 2, 5], [1, 3, 2, 37]]


def test_empty_and_another_stream():
    from fovi_b200 import tokens
    x, pos, f = _inputs(2, 10, 4, 64, (16, 16), 0, True, BF, 4)
    assert tokens.rotary(x[:0], pos, f, (16, 16)).shape == (0, 10, 4, 64)
    assert tokens.rotary(x[:, :0], pos[:0], f, (16, 16)).shape == (2, 0, 4, 64)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = tokens.rotary(x, pos, f, (16, 16))
    torch.cuda.current_stream().wait_stream(stream)
    oracle.near(y, oracle.rotary(x, pos, f, (16, 16)))


def test_module():
    """Frequencies as documented, float32 whatever the model is cast to, and not part of the state dict."""
    from fovi_b200.tokens import AxialRotary
    m = AxialRotary(64, axes=3, units=[1.0, 2 * math.pi, 2 * math.pi]).to(torch.bfloat16)
    assert m.pairs_per_axis == (11, 11, 10) and m.frequencies.dtype is torch.float32 and m.frequencies.is_cuda and not m.state_dict()
    want = [u * 100.0 ** (-j / n) for u, n in ((1.0, 11), (2 * math.pi, 11), (2 * math.pi, 10)) for j in range(n)]
    assert torch.equal(m.frequencies.cpu(), torch.tensor(want, dtype=torch.float32))
    x, pos, _ = _inputs(2, 12, 4, 64, (11, 11, 10), 1, False, BF, 9)
    oracle.near(m(x, pos, prefix=1), oracle.rotary(x, pos, m.frequencies, (11, 11, 10), 1))


@pytest.mark.autograd
def test_refusals():
    from fovi_b200 import tokens
    x, pos, f = _inputs(2, 10, 4, 64, (16, 16), 0, True, F32, 4)
    with pytest.raises(ValueError, match="CUDA"):
        tokens.rotary(x.cpu(), pos, f, (16, 16))
    with pytest.raises(ValueError, match="shape"):
        tokens.rotary(x[0], pos, f, (16, 16))
    with pytest.raises(ValueError, match="pairs_per_axis"):
        tokens.rotary(x, pos, f, (17, 16))
    with pytest.raises(ValueError, match="pairs_per_axis"):
        tokens.rotary(x, pos, f, (8, 8, 8, 4, 4))
    with pytest.raises(ValueError, match="pairs_per_axis"):
        tokens.rotary(x, pos, f, (-1, 33))
    with pytest.raises(ValueError, match="frequencies"):
        tokens.rotary(x, pos, f[:31], (16, 16))
    with pytest.raises(ValueError, match="positions"):
        tokens.rotary(x, pos, f, (16, 16), prefix=1)
    with pytest.raises(ValueError, match="prefix"):
        tokens.rotary(x, pos, f, (16, 16), prefix=11)
    with pytest.raises(ValueError, match="pairing"):
        tokens.rotary(x, pos, f, (16, 16), pairing="thirds")
    with pytest.raises(TypeError, match="float32"):
        tokens.rotary(x, pos.double(), f, (16, 16))
    with pytest.raises(TypeError, match="dtype"):
        tokens.rotary(x.half(), pos, f, (16, 16))
    with pytest.raises(NotImplementedError, match="no gradient"):
        tokens.rotary(x, pos.requires_grad_(True), f, (16, 16))
