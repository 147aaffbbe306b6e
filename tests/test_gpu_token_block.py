"""GPU: a token block's operators together: FixationReader with feed-forward halves, a block served in 8 bits, both inside captured graphs, and the products' failure path."""
import pytest
import torch
import torch.nn.functional as F

from oracle import block_oracle as oracle
from test_gpu_fixation_reader import _images, _reader

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
FOVI_ERR_DEVICE_TIMEOUT = 6   # include/fovi_b200.h


def _with_feed_forward(hidden, **kw):
    """The reader of test_gpu_fixation_reader, whose blocks get a feed-forward half."""
    from fovi_b200.tokens import FixationReader
    base = _reader(**kw)
    torch.manual_seed(11)
    m = FixationReader(base.retina, base.embedding, base.dim, base.blocks[0].heads, 10, queries=base.queries.shape[0], depth=len(base.blocks), feed_forward=hidden).cuda()
    missing, unexpected = m.load_state_dict(base.state_dict(), strict=False)
    assert not unexpected and missing and all(k.startswith("feed_forward") for k in missing)
    for n in m.feed_forward_norms:
        n.weight.data.uniform_(0.5, 1.5)
    return m


def _plain_read(m, states, places):
    """m.read in 64 bits."""
    lin = lambda l, x: F.linear(x, l.weight.double(), l.bias.double())  # noqa: E731
    norm = lambda n, x: F.layer_norm(x, x.shape[-1:], n.weight.double(), n.bias.double(), n.eps)  # noqa: E731
    states, places, P = states.double(), places.double(), m.rotary.frequencies.numel()
    axis = [a for a, n in enumerate(m.rotary.pairs_per_axis) for _ in range(n)]
    t = (places[..., axis] * m.rotary.frequencies.double())[:, :, None]
    x = m.queries.double().expand(states.shape[0], -1, -1)
    for n, b, rn, ff in zip(m.norms, m.blocks, m.feed_forward_norms, m.feed_forwards):
        q = lin(b.query, norm(n, x)).unflatten(-1, (b.heads, -1))
        k, v = (lin(l, states).unflatten(-1, (b.kv_heads, -1)) for l in (b.key, b.value))
        u, w, rest = k[..., :P], k[..., P:2 * P], k[..., 2 * P:]
        k = torch.cat([u * t.cos() - w * t.sin(), w * t.cos() + u * t.sin(), rest], -1)
        s = torch.einsum("bqhd,bkhd->bhqk", q, k) * b.head_dim ** -0.5
        x = x + lin(b.out, torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v).flatten(2))
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + rn.eps) * rn.weight.double()
        x = x + lin(ff.down, F.silu(lin(ff.gate, y)) * lin(ff.up, y))
    return lin(m.classifier, norm(m.norm, x).mean(1))


@pytest.mark.autograd
def test_reading_and_its_gradients():
    """float32: scores and every parameter's gradient against the same in 64 bits.  Two blocks, of ten float32 products each and their gradients, each of up to 2 (n + 8) half-units for
    sums of n = 1100 terms, in the worst case 2e-3 of a gradient's size; what roundings that do not conspire give is a hundredth of that, and is asked for."""
    m = _with_feed_forward(250)
    images, fix = _images()
    with torch.no_grad():
        states, places = m.states(images, fix)
    states = states.float()
    params = [p for n, p in m.named_parameters() if not n.startswith(("embedding", "retina", "state_norm"))]
    target = torch.tensor([1, 5, 7], device="cuda")
    got = m.read(states, places)
    want = _plain_read(m, states, places)
    g = torch.autograd.grad(F.cross_entropy(got, target), params)
    w = torch.autograd.grad(F.cross_entropy(want, target), params)
    assert torch.linalg.vector_norm(got.double() - want) <= 2e-5 * torch.linalg.vector_norm(want)
    for a, b in zip(g, w, strict=True):
        assert torch.linalg.vector_norm(a.double() - b) <= 2e-5 * torch.linalg.vector_norm(b) + 1e-9


@pytest.mark.autograd
def test_without_it_nothing_changes():
    m = _reader()
    assert not any(k.startswith("feed_forward") for k in m.state_dict())
    with torch.no_grad():
        images, fix = _images()
        assert m(images, fix).shape == (3, 10)


@pytest.mark.autograd
def test_under_autocast():
    """bf16 products around a float32 stream: as near to float32 as bf16 lets two blocks be, and every parameter has a gradient of its own type."""
    m = _with_feed_forward(256)
    images, fix = _images()
    with torch.no_grad():
        plain = m(images, fix)
    with torch.autocast("cuda", torch.bfloat16):
        y = m(images, fix)
    assert torch.linalg.vector_norm(y.float() - plain) <= 0.05 * torch.linalg.vector_norm(plain)
    y.float().square().sum().backward()
    for name, p in m.named_parameters():
        assert p.grad is not None and p.grad.dtype is p.dtype and torch.isfinite(p.grad).all(), name


def _serving(C, hidden, dtype):
    """A block's second half in 8 bits: norm, one layer to twice the hidden channels, the gate, one layer back."""
    from fovi_b200 import tokens
    torch.manual_seed(C)
    up, down = tokens.Linear8(torch.nn.Linear(C, 2 * hidden, device="cuda"), dtype), tokens.Linear8(torch.nn.Linear(hidden, C, device="cuda"), dtype)
    norm = tokens.TokenRMSNorm(C)

    def step(x, stream):
        q, scale, stream = tokens.rms_norm_int8(x, norm.weight, residual=stream)
        g, u = up(q, scale).chunk(2, -1)
        return down(F.silu(g) * u), stream
    return step, up, down, norm


@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("rows", [1, 20, 300])
def test_served_in_eight_bits(rows, dtype):
    """Every stage against the stage in 64 bits, on what the one before gave."""
    from fovi_b200 import tokens
    step, up, down, norm = _serving(136, 260, dtype)
    x, stream = (torch.randn(rows, 136, device="cuda").to(dtype) for _ in range(2))
    y, total = step(x, stream)
    assert torch.equal(total, x + stream)
    q, scale, _ = tokens.rms_norm_int8(x, norm.weight, residual=stream)
    value = oracle.rms_norm(x, norm.weight, 1e-6, stream)[0][0]
    oracle.near_eight_bits(q, scale, value, value.abs() * 156 * oracle.U32)
    h = up(q, scale)
    oracle.near(h, oracle.linear_int8(q, scale, up.weight, up.weight_scale, up.bias, dtype))
    g, u = h.chunk(2, -1)
    q, scale = tokens.quantize(F.silu(g) * u)
    oracle.near(y, oracle.linear_int8(q, scale, down.weight, down.weight_scale, down.bias, dtype))


def _captured(step):
    """step's captured graph and its result."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


@pytest.mark.parametrize("rows", [1, 33, 300])
def test_serving_captured_and_replayed(rows):
    """Two graphs of one block, replayed in turn: each has memory of its own."""
    from fovi_b200 import tokens
    step, *_ = _serving(136, 260, BF)
    ff = tokens.GatedFeedForward(136, 264, dtype=BF)
    x, stream = (torch.randn(rows, 136, device="cuda", dtype=BF) for _ in range(2))

    def both():
        y, total = step(x, stream)
        return ff(y) + total, total
    graphs = [_captured(both) for _ in range(2)]
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        want = both()
        for graph, out in graphs:
            for t in out:
                t.zero_()
            graph.replay()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    tokens.check()


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("rows", [5, 300])
def test_training_captured_and_replayed(rows, dtype):
    from fovi_b200 import tokens
    g = torch.Generator(device="cuda").manual_seed(rows)
    def n(*s, scale=1.0): return (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype).requires_grad_(True)
    x, res, w, wg, wu, wd, b = n(rows, 96), n(rows, 96), n(96), n(136, 96, scale=0.1), n(136, 96, scale=0.1), n(96, 136, scale=0.1), n(96)
    leaves = (x, res, w, wg, wu, wd, b)

    def step():
        y, total = tokens.rms_norm(x, w, residual=res)
        out = tokens.gated_feed_forward(y, wg, wu, wd, down_bias=b) + total
        return (out.detach(),) + torch.autograd.grad(out, leaves, out.detach())
    graph, got = _captured(step)
    for _ in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        want = step()
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    tokens.check()


def test_a_wait_that_gives_up():
    """A product whose loads are withheld reports so on the host, nothing faults, and the next call is right."""
    from fovi_b200 import ops, tokens
    from fovi_b200._lib import FoviError, check, lib
    q, w = (torch.randint(-128, 128, (n, 320), device="cuda", dtype=torch.int8) for n in (300, 200))
    s, ws = torch.rand(300, device="cuda"), torch.rand(200, device="cuda")
    y = torch.empty(300, 200, device="cuda", dtype=BF)
    tokens.check()
    check(lib.fovi_linear_int8_selftest_wait_timeout(q.data_ptr(), 300, 320, 320, s.data_ptr(), w.data_ptr(), 200, 320, ws.data_ptr(), None, y.data_ptr(), ops.BF16, ops._stream()), "selftest")
    with pytest.raises(FoviError, match="wait site") as e:
        tokens.check()
    assert e.value.status == FOVI_ERR_DEVICE_TIMEOUT
    tokens.check()                                # cleared by the failing check
    oracle.near(tokens.linear_int8(q, s, w, ws), oracle.linear_int8(q, s, w, ws, None, BF))
    tokens.check()


def test_unaligned_pointers_are_refused_by_the_c_abi():
    from fovi_b200 import ops
    from fovi_b200._lib import lib
    b = torch.zeros(4096, device="cuda", dtype=BF)
    p, st = b.data_ptr(), ops._stream()
    args = [p, ops.BF16, 4, 16, 16, 16, 16, p, 16, p, 16, p, 16, None, None, None, 0, p, None, p, 4096, st]
    for i in (17, 19):                                                          # y, work
        bad = list(args)
        bad[i] = p + 8
        assert lib.fovi_gated_ffn_forward(*bad) == 5
    for i, v in ((0, p + 2), (7, p + 2), (9, p + 2), (11, p + 2), (6, 17), (8, 17), (10, 17), (12, 17), (20, 8)):      # rows off boundaries: more work is needed than is there
        bad = list(args)
        bad[i], bad[20] = v, lib.fovi_gated_ffn_workspace_bytes(ops.BF16, 4, 16, 16, 16, 0) - (i == 20)
        assert lib.fovi_gated_ffn_forward(*bad) == 1
    for i, v in ((1, 5), (2, -1), (3, 0), (4, 0), (5, 0), (6, -1), (16, 2), (16, -1), (0, None), (17, None), (19, None)):
        bad = list(args)
        bad[i] = v
        assert lib.fovi_gated_ffn_forward(*bad) == 1
    assert lib.fovi_gated_ffn_workspace_bytes(ops.BF16, 4, 16, 16, 16, 3) == -1 == lib.fovi_gated_ffn_workspace_bytes(ops.BF16, 4, 16, 16, 16, 7)
    assert lib.fovi_linear_int8(p + 1, 4, 16, 16, p, p, 16, 16, p, None, p, 0, st) == 5
    assert lib.fovi_linear_int8(p, 4, 16, 17, p, p, 16, 16, p, None, p, 0, st) == 5
    assert lib.fovi_linear_int8(p, 4, 131072, 131072, p, p, 16, 131072, p, None, p, 0, st) == 1


@pytest.mark.autograd
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("rows", [5, 700])
def test_three_streams_at_once(rows, dtype):
    """Calls that run beside one another give the bits that they give alone."""
    from fovi_b200 import tokens

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        def n(*s, scale=1.0): return (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype).requires_grad_(True)
        return [n(rows, 96), n(rows, 96), n(96), n(344, 96, scale=0.1), n(344, 96, scale=0.1), n(96, 344, scale=0.1)]

    def step(t):
        y, total = tokens.rms_norm(t[0], t[2], residual=t[1])
        out = tokens.gated_feed_forward(y, *t[3:]) + total
        with torch.no_grad():
            eight = tokens.linear_int8(*tokens.rms_norm_int8(t[0], t[2]), *tokens.quantize(t[3]))
        return [out, eight, *torch.autograd.grad(out, t, out.detach())]
    sets = [inputs(i) for i in range(3)]
    want = [step(t) for t in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for stream, t in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(step(t))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for a, b in zip(got, want) for p, q in zip(a, b))
    tokens.check()
