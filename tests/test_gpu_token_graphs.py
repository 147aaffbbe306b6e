"""GPU: the token operators inside a captured graph, as a serving loop replays them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_and_replayed(dtype):
    from fovi_b200 import tokens
    B, Lk, H, D = 3, 700, 6, 64
    x, w, b = torch.randn(B, 1, H * D, device="cuda").to(dtype), torch.rand(H * D, device="cuda"), torch.rand(H * D, device="cuda")
    k, v = (torch.randn(B, Lk, H, D, device="cuda").to(dtype) for _ in range(2))
    pos, f = torch.rand(B, 1, 2, device="cuda"), torch.rand(32, device="cuda")
    lengths = torch.full((B,), Lk, dtype=torch.int32, device="cuda")

    def step():
        q = tokens.rotary(tokens.layer_norm(x, w, b).view(B, 1, H, D), pos, f, (16, 16))
        return tokens.cross_attention(q, k, v, key_lengths=lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in (700, 1, 0, 333):
        x.copy_(torch.randn_like(x))
        pos.copy_(torch.rand_like(pos))
        lengths.fill_(n)
        graph.replay()
        assert torch.equal(out, step())
    tokens.check()
