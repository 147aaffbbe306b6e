"""GPU: key_lengths of cross attention in every whole-number type, where the number of keys is more than the type holds too."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
@pytest.mark.parametrize("Lk", [50, 300, 40000])
def test_types(Lk, dtype):
    from fovi_b200 import tokens
    q, k, v = (torch.randn(4, n, 2, 64, device="cuda", dtype=torch.bfloat16) for n in (3, Lk, Lk))
    lengths = [0, 1, 77, 127]
    want = tokens.cross_attention(q, k, v, key_lengths=torch.tensor([min(n, Lk) for n in lengths], dtype=torch.int32, device="cuda"))
    assert torch.equal(tokens.cross_attention(q, k, v, key_lengths=torch.tensor(lengths, dtype=dtype, device="cuda")), want)


def test_beyond_both_ends():
    """Taken into 0 .. Lk, also from numbers that 32 bits do not hold."""
    from fovi_b200 import tokens
    q, k, v = (torch.randn(4, n, 2, 64, device="cuda", dtype=torch.bfloat16) for n in (3, 90, 90))
    want = tokens.cross_attention(q, k, v, key_lengths=torch.tensor([0, 90, 0, 90], dtype=torch.int32, device="cuda"))
    assert torch.equal(tokens.cross_attention(q, k, v, key_lengths=torch.tensor([-5, 91, -2 ** 40 + 7, 2 ** 40 + 7], device="cuda")), want)
