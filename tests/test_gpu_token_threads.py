"""GPU: token operators called from several threads at once, each in its first call of that width."""
from concurrent.futures import ThreadPoolExecutor
from threading import Barrier

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [52, 300, 516, 1100, 2052, 4100])
def test_first_calls_at_once(width):
    from fovi_b200 import tokens
    x = [torch.randn(700, width, device="cuda") for _ in range(8)]
    ready = Barrier(8)

    def work(t):
        with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
            ready.wait()
            got = tokens.rms_norm(t), tokens.layer_norm(t), tokens.quantize(t), tokens.rms_norm(t.bfloat16()), tokens.layer_norm(t.bfloat16())
            torch.cuda.current_stream().synchronize()
            return got
    torch.cuda.synchronize()
    with ThreadPoolExecutor(8) as pool:
        got = list(pool.map(work, x))
    for t, (rms, norm, (q, s), *halves) in zip(x, got):
        assert torch.equal(rms, tokens.rms_norm(t)) and torch.equal(norm, tokens.layer_norm(t))
        assert torch.equal(q, tokens.quantize(t)[0]) and torch.equal(s, tokens.quantize(t)[1])
        assert torch.equal(halves[0], tokens.rms_norm(t.bfloat16())) and torch.equal(halves[1], tokens.layer_norm(t.bfloat16()))
