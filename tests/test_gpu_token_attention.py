"""GPU: cross attention and its gradients against the definition in 64 bits, on the kernels that the shape and the type choose."""
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


def _inputs(B, Lq, Lk, H, Hkv, D, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v, dy = (torch.randn(shape, generator=g, device="cuda").to(dtype) for shape in ((B, Lq, H, D), (B, Lk, Hkv, D), (B, Lk, Hkv, D), (B, Lq, H, D)))
    return q, k, v, dy


def _check(q, k, v, dy, **mask):
    from fovi_b200 import tokens
    q, k, v = leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = tokens.cross_attention(q, k, v, **mask)
    assert o.dtype is q.dtype and o.is_contiguous()
    got = (o.detach(),) + torch.autograd.grad(o, leaves, dy)
    for g, want in zip(got, oracle.attention(q.detach(), k.detach(), v.detach(), dy=dy, **mask)):
        oracle.near(g, want)
    with torch.no_grad():
        assert torch.equal(tokens.cross_attention(q, k, v, **mask), o)
    tokens.check()
    return got


SHAPES = [  # B, Lq, Lk, H, Hkv, D
    (1, 1, 1, 1, 1, 1), (1, 1, 1, 1, 1, 64), (2, 1, 65, 6, 6, 64), (2, 1, 2056, 4, 4, 64), (1, 3, 7, 2, 1, 8), (2, 65, 65, 6, 6, 64), (1, 257, 300, 2, 2, 64),
    (1, 128, 128, 2, 1, 128), (1, 129, 127, 4, 2, 128), (2, 16, 261, 6, 3, 64), (1, 100, 129, 8, 1, 32), (1, 130, 1030, 2, 2, 80), (3, 7, 64, 5, 5, 96), (1, 40, 70, 3, 3, 40),
    (1, 33, 77, 2, 2, 7), (2, 5, 200, 2, 2, 63), (1, 256, 512, 1, 1, 64), (1, 1, 3000, 16, 4, 128), (1, 8, 5000, 2, 1, 64), (2, 64, 1, 2, 2, 64), (1, 600, 33, 1, 1, 64),
    (2, 2, 130, 12, 2, 64), (1, 31, 4100, 4, 1, 16)]


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(shape, dtype):
    _check(*_inputs(*shape, dtype, sum(shape)))


def test_many_blocks_of_few_queries():
    """Warps without a query do no arithmetic and would run ahead of the one that does; several blocks follow one another on every SM."""
    from fovi_b200 import tokens
    for B, Lq, Lk, D in ((64, 1, 2056, 64), (40, 33, 700, 128), (64, 70, 1030, 64)):
        q, k, v, _ = _inputs(B, Lq, Lk, 20, 20, D, BF, Lk)
        for kw in ({}, dict(key_lengths=torch.randint(0, Lk + 1, (B,), device="cuda", dtype=torch.int32)), dict(key_mask=torch.rand(B, Lk, device="cuda") < 0.7)):
            got = tokens.cross_attention(q, k, v, **kw)
            tokens.check()
            for b in range(0, B, 8):
                part = {n: t[b:b + 8] for n, t in kw.items()}
                oracle.near(got[b:b + 8], oracle.attention(q[b:b + 8], k[b:b + 8], v[b:b + 8], **part))


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D,H,Hkv", [(64, 4, 4), (128, 4, 2), (80, 2, 1), (7, 2, 2)])
@pytest.mark.parametrize("Lq,Lk", [(1, 300), (70, 300), (5, 129), (140, 64)])
def test_masks(Lq, Lk, D, H, Hkv, dtype):
    """Lengths of zero, one, one tile, one more, all and beyond; keys dropped at random, whole tiles of them, all of a sample's; both together."""
    B = 7
    q, k, v, dy = _inputs(B, Lq, Lk, H, Hkv, D, dtype, Lq + Lk + D)
    lengths = torch.tensor([0, 1, 64, 65, Lk - 1, Lk, Lk + 50], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    mask = torch.rand((B, Lk), generator=g, device="cuda") < 0.7
    mask[2] = False
    mask[3, :128] = False
    mask[4, 1:] = False
    mask[5, 100:] = False
    for kw in (dict(key_lengths=lengths), dict(key_mask=mask), dict(key_lengths=lengths, key_mask=mask)):
        _check(q, k, v, dy, **kw)


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128, 24])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_what_masked_keys_hold_has_no_effect(junk, D, dtype):
    B, Lq, Lk, H = 3, 67, 200, 2
    q, k, v, dy = _inputs(B, Lq, Lk, H, H, D, dtype, 5)
    lengths = torch.tensor([0, 77, 200], dtype=torch.int64, device="cuda")
    mask = torch.rand((B, Lk), device="cuda") < 0.8
    hidden = (torch.arange(Lk, device="cuda") >= lengths[:, None]) | ~mask
    clean = _check(q, k, v, dy, key_lengths=lengths, key_mask=mask)
    kj, vj = (torch.where(hidden[:, :, None, None], torch.tensor(junk, dtype=dtype, device="cuda"), t) for t in (k, v))
    from fovi_b200 import tokens
    leaves = [t.detach().requires_grad_(True) for t in (q, kj, vj)]
    o = tokens.cross_attention(*leaves, key_lengths=lengths, key_mask=mask)
    for a, b in zip(clean, (o.detach(),) + torch.autograd.grad(o, leaves, dy)):
        assert torch.equal(a, b)
    assert not o[0].any()


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
def test_not_a_number_stays_in_its_row(dtype):
    """A query that is not a number reaches its own row and the gradients of the keys that it reads; one whose sample has no key reaches nothing."""
    from fovi_b200 import tokens
    q, k, v, dy = _inputs(2, 70, 140, 2, 2, 64, dtype, 5)
    q[:, 3, 1, 7] = float("nan")
    lengths = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = tokens.cross_attention(*leaves, key_lengths=lengths)
    gq, gk, gv = torch.autograd.grad(o, leaves, dy)
    assert not o[0].any() and not gq[0].any() and not gk[0].any() and not gv[0].any()
    bad = torch.isnan(o)
    assert bad[1, 3, 1].all() and bad.sum() == 64
    assert torch.isnan(gk[1, :100, 1]).all() and not torch.isnan(gk[:, :, 0]).any() and not gk[1, 100:].any() and not gv[1, 100:].any()


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_strides(D, dtype):
    """Heads in front of tokens, slices of packed projections, a start on no 16-byte boundary, channels apart, expanded queries and states, a strided and an expanded gradient."""
    B, Lq, Lk, H = 2, 35, 150, 4
    q, k, v, dy = _inputs(B, Lq, Lk, H, H, D, dtype, 11)
    def front(t): return t.transpose(1, 2).contiguous().transpose(1, 2)
    kv = torch.randn(B, Lk, 2, H, D, device="cuda").to(dtype)
    off = torch.randn(B, Lk, H, D + 1, device="cuda").to(dtype)[..., 1:]
    apart = k.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    for a, b, c, g in ((front(q), front(k), front(v), front(dy)), (q, kv[:, :, 0], kv[:, :, 1], dy), (q, off, v, dy), (q, apart, apart, dy),
                       (q[:1].expand(B, -1, -1, -1), k, v, dy), (q, k[:1].expand(B, -1, -1, -1), v[:, :, :1].expand(-1, -1, H, -1), dy),
                       (q, k[:, ::1], v, dy[:, :1].expand(-1, Lq, -1, -1)), (q[:, :, ::2], k[:, :, ::2], v[:, :, 1::2], dy[:, :, ::2])):
        _check(a, b, c, g)
    from fovi_b200 import tokens
    shared = torch.randn(Lq, H, D, device="cuda").to(dtype).requires_grad_(True)         # learned queries, one set for all samples
    o = tokens.cross_attention(shared.expand(B, -1, -1, -1), k, v)
    gq, = torch.autograd.grad(o.sum(), shared)
    want = oracle.attention(shared.detach().expand(B, -1, -1, -1), k, v, dy=torch.ones_like(dy))[1]
    value, bound = want[0].sum(0), want[1].sum(0)
    oracle.near(gq, (value, bound + 2 * (oracle.U16 if dtype is BF else oracle.U32) * (want[0].abs().sum(0) + bound)))


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales(scale, dtype):
    """No scale at all (the mean of the states), a negative one, and one so large that a row is one key."""
    _check(*_inputs(2, 66, 190, 2, 2, 64, dtype, 17), scale=scale)


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [0.0, -0.3, -4.0])
def test_scales_with_masks(scale, dtype):
    """A masked score has to lose whatever the scale's sign, and without a scale; what the masked states hold stays out."""
    q, k, v, dy = _inputs(3, 66, 290, 2, 1, 64, dtype, 23)
    mask = torch.rand(3, 290, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") < 0.6
    mask[1] = False
    kw = dict(key_mask=mask, key_lengths=torch.tensor([290, 290, 129], dtype=torch.int32, device="cuda"), scale=scale)
    want = _check(q, k, v, dy, **kw)
    from fovi_b200 import tokens
    gone = ~mask | (torch.arange(290, device="cuda") >= kw["key_lengths"][:, None])
    k, v = (t.masked_fill(gone[:, :, None, None], float("nan")).requires_grad_(True) for t in (k, v))
    q = q.requires_grad_(True)
    o = tokens.cross_attention(q, k, v, **kw)
    for g, w in zip((o,) + torch.autograd.grad(o, (q, k, v), dy), want):
        assert torch.equal(g, w)


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rising_scores(dtype):
    """Keys whose scores rise by hundreds from tile to tile, so that the running maximum moves in every one; and fall."""
    q, k, v, dy = _inputs(1, 40, 700, 1, 1, 64, dtype, 3)
    q = q.abs()
    ramp = torch.linspace(-2, 2, 700, device="cuda").to(dtype)[None, :, None, None]
    for r in (ramp, ramp.flip(1)):
        _check(q, (k * 0.05 + r).to(dtype), v, dy, scale=0.5)


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Lk", [1, 90])
def test_one_key_has_weight_one(Lk, D, dtype):
    """Its gradients with respect to the score's sides are zeros, not what roundings leave of them."""
    q, k, v, dy = _inputs(3, 70, Lk, 2, 2, D, dtype, 8)
    o, gq, gk, gv = _check(q, k, v, dy, key_lengths=torch.ones(3, dtype=torch.int32, device="cuda"))
    assert torch.equal(o, v[:, :1].expand_as(o)) and not gq.any() and not gk.any() and not gv[:, 1:].any()


@pytest.mark.autograd
def test_delta_of_few_keys():
    """bf16: where a row's weight lies on a key or two, the rounding of the result is not to be seen in dq and dk: their error is that of two roundings to bf16 of independent values, as where
    it lies on many.  (2^-9 / sqrt(3) of the value at most, each, in the root mean square; 1.1 for what is not rounded there.)"""
    from fovi_b200 import ops
    for Lk in (2, 3, 6, 40):
        q, k, v, dy = _inputs(4, 200, Lk, 4, 4, 64, BF, Lk)
        o, lse = ops.attention(q, k, v, want_lse=True)
        for got, (want, _) in zip(ops.attention_backward(q, k, v, o, dy, lse)[:2], oracle.attention(q, k, v, dy=dy)[1:3]):
            assert (got.double() - want).norm() <= 1.1 * 2 ** 0.5 * 2.0 ** -8 / 3 ** 0.5 * want.norm()


@pytest.mark.autograd
def test_no_keys_no_queries_no_samples():
    from fovi_b200 import tokens
    for B, Lq, Lk in ((2, 5, 0), (2, 0, 5), (0, 5, 5)):
        q, k, v, dy = _inputs(B, Lq, Lk, 2, 2, 64, BF, 1)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        o = tokens.cross_attention(*leaves)
        grads = torch.autograd.grad(o, leaves, dy)
        assert o.shape == q.shape and not o.any()
        assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, leaves))


@pytest.mark.autograd
def test_gradients_that_are_wanted():
    """Each input alone: the others' gradients are not made."""
    from fovi_b200 import tokens
    for dtype in (BF, F32):
        q, k, v, dy = _inputs(2, 20, 90, 2, 2, 64, dtype, 2)
        want = oracle.attention(q, k, v, dy=dy)
        for i in range(3):
            leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
            g, = torch.autograd.grad(tokens.cross_attention(*leaves), leaves[i], dy)
            oracle.near(g, want[1 + i])


def test_same_bits_every_time():
    from fovi_b200 import ops
    for shape in ((2, 70, 300, 4, 2, 64), (1, 1, 3000, 4, 4, 64), (1, 8, 700, 2, 2, 128)):
        for dtype in (BF, F32):
            q, k, v, dy = _inputs(*shape, dtype, 4)
            o, lse = ops.attention(q, k, v, want_lse=True)
            first = (o, lse) + ops.attention_backward(q, k, v, o, dy, lse)
            for _ in range(3):
                o2, lse2 = ops.attention(q, k, v, want_lse=True)
                assert all(torch.equal(a, b) for a, b in zip(first, (o2, lse2) + ops.attention_backward(q, k, v, o2, dy, lse2)))


@pytest.mark.autograd
def test_another_stream():
    stream = torch.cuda.Stream()
    for dtype in (BF, F32):
        args = _inputs(2, 70, 300, 4, 2, 64, dtype, 4)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            _check(*args)
        torch.cuda.current_stream().wait_stream(stream)


def test_states_whose_offsets_pass_32_bits():
    """A view whose last sample starts more than 2^32 elements behind the first: 9 GB, of which two samples are read."""
    from fovi_b200 import ops
    Lk, H, D = 300, 2, 64
    gap = (1 << 32) + 4096
    store = torch.empty(gap + 2 * Lk * H * D, dtype=BF, device="cuda")
    k = store.as_strided((2, Lk, H, D), (gap, H * D, D, 1))
    q, kk, v, _ = _inputs(2, 5, Lk, H, H, D, BF, 6)
    k.copy_(kk)
    for rows in (1, 5):
        oracle.near(ops.attention(q[:, :rows], k, v), oracle.attention(q[:, :rows], kk, v))
    k32 = store.view(torch.float32).as_strided((2, Lk, H, D), (gap // 2, H * D, D, 1))
    k32.copy_(kk)
    oracle.near(ops.attention(q.float(), k32, v.float()), oracle.attention(q.float(), kk.float(), v.float()))


def test_gradient_against_differences():
    """Central differences of the float32 kernel's own forward pass along a random direction; the difference between two step sizes bounds the truncation."""
    from fovi_b200 import ops
    q, k, v, dy = _inputs(1, 9, 70, 2, 1, 16, F32, 21)
    lengths = torch.tensor([66], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    o, lse = ops.attention(q, k, v, lengths, want_lse=True)
    grads = ops.attention_backward(q, k, v, o, dy, lse, lengths)
    for i, t in enumerate((q, k, v)):
        d = torch.randn(t.shape, generator=g, device="cuda")
        def loss(h):
            args = [a + h * d if j == i else a for j, a in enumerate((q, k, v))]
            return (ops.attention(*args, lengths).double() * dy.double()).sum().item()
        near, far = ((loss(h) - loss(-h)) / (2 * h) for h in (2.0 ** -7, 2.0 ** -6))
        bound = oracle.attention(q, k, v, lengths)[1]
        rounding = 2 * (bound * dy.double().abs()).sum().item() / (2 * 2.0 ** -7)
        assert abs((grads[i].double() * d.double()).sum().item() - near) <= abs(near - far) + rounding


def test_refusals():
    from fovi_b200 import tokens
    from fovi_b200.tokens import CrossAttention
    q, k, v, _ = _inputs(2, 5, 9, 4, 2, 64, F32, 1)
    with pytest.raises(ValueError, match="CUDA"):
        tokens.cross_attention(q.cpu(), k, v)
    with pytest.raises(ValueError, match="wanted"):
        tokens.cross_attention(q, k, v[:, :8])
    with pytest.raises(ValueError, match="wanted"):
        tokens.cross_attention(q[0], k, v)
    with pytest.raises(ValueError, match="wanted"):
        tokens.cross_attention(q[:1], k, v)
    with pytest.raises(ValueError, match="share"):
        tokens.cross_attention(q[:, :, :3], k, v)
    with pytest.raises(ValueError, match="channels"):
        tokens.cross_attention(*(torch.zeros(1, 2, 1, 136, device="cuda") for _ in range(3)))
    with pytest.raises(TypeError, match="one type"):
        tokens.cross_attention(q, k.bfloat16(), v)
    with pytest.raises(TypeError, match="dtype"):
        tokens.cross_attention(q.half(), k.half(), v.half())
    with pytest.raises(ValueError, match="key_lengths"):
        tokens.cross_attention(q, k, v, key_lengths=torch.ones(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="key_lengths"):
        tokens.cross_attention(q, k, v, key_lengths=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="key_mask"):
        tokens.cross_attention(q, k, v, key_mask=torch.ones(2, 9, device="cuda"))
    with pytest.raises(ValueError, match="key_mask"):
        tokens.cross_attention(q, k, v, key_mask=torch.ones(2, 8, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError, match="scale"):
        tokens.cross_attention(q, k, v, scale=float("inf"))
    with pytest.raises(ValueError, match="divide"):
        CrossAttention(100, 3)
