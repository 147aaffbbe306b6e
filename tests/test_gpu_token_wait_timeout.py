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


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("states", [False, True])
def test_backward(D, states):
    """dq alone, and dk and dv alone."""
    from fovi_b200 import ops, tokens
    from fovi_b200._lib import FoviError, check, lib
    q, k, v, dy = (torch.randn(2, n, 3, D, device="cuda", dtype=torch.bfloat16) for n in (150, 300, 300, 150))
    o, lse = ops.attention(q, k, v, want_lse=True)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    size = lib.fovi_attention_workspace_bytes(1, 2, 150, 300, 3, 3, D, 1)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    ptr = [g.data_ptr() if states == (i > 0) else None for i, g in enumerate(grads)]
    tokens.check()
    check(lib.fovi_attention_backward_selftest_wait_timeout(*(t.data_ptr() for t in (q, k, v, o, dy)), 2, 150, 300, 3, 3, D,
                                                            ops._I64x12(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *dy.stride()[:3]), D ** -0.5, lse.data_ptr(), *ptr,
                                                            work.data_ptr(), size, ops._stream()), "selftest")
    with pytest.raises(FoviError, match="wait site") as e:
        tokens.check()
    assert e.value.status == FOVI_ERR_DEVICE_TIMEOUT
    tokens.check()
    for got, want in zip(ops.attention_backward(q, k, v, o, dy, lse), oracle.attention(q, k, v, dy=dy)[1:]):
        oracle.near(got, want)
    tokens.check()
