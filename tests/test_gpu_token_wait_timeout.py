"""GPU: the failure path of the tensor-core attention kernels.  A wait that runs out surfaces as a status that the host reads, nothing faults, and the next call is right.
The wait is made to run out by a diagnostic launch that withholds its loads and waits for a few thousand attempts."""
import pytest
import torch

from oracle import token_oracle as oracle

pytestmark = pytest.mark.gpu
FOVI_ERR_DEVICE_TIMEOUT = 6   # include/fovi_b200.h


@pytest.mark.parametrize("D", [64, 128])
def test_forward(D):
    from fovi_b200 import ops, tokens
    from fovi_b200._lib import FoviError, check, lib
    q, k, v = (torch.randn(2, n, 3, D, device="cuda", dtype=torch.bfloat16) for n in (150, 300, 300))
    o = torch.empty_like(q)
    tokens.check()
    check(lib.fovi_attention_forward_selftest_wait_timeout(q.data_ptr(), k.data_ptr(), v.data_ptr(), 2, 150, 300, 3, 3, D,
                                                           ops._I64x9(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3]), 0.125, o.data_ptr(), ops._stream()), "selftest")
    with pytest.raises(FoviError, match="wait site") as e:
        tokens.check()
    assert e.value.status == FOVI_ERR_DEVICE_TIMEOUT
    tokens.check()                                # cleared by the failing check
    oracle.near(tokens.cross_attention(q, k, v), oracle.attention(q, k, v))
    tokens.check()
