"""CPU: sizes that depend on a device's SMs are asked for with the tensors' device as the current one, as the launch is."""
import contextlib

import pytest
import torch


@pytest.fixture
def asked(monkeypatch):
    """Names of the library's functions called, with the device that was current."""
    from fovi_b200 import ops
    calls, current = [], [None]

    @contextlib.contextmanager
    def on(device):
        before, current[0] = current[0], device
        yield
        current[0] = before

    class Lib:
        def __getattr__(self, name):
            def call(*args):
                calls.append((name, current[0]))
                return 64 if name.endswith("_bytes") else 0
            return call
    monkeypatch.setattr(ops, "lib", Lib())
    monkeypatch.setattr(ops, "_on", on)
    monkeypatch.setattr(ops, "_need_cuda", lambda *a: None)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    return calls


def _meta(*s, dtype=torch.float32):
    return torch.empty(*s, dtype=dtype, device="meta")


def _check(calls, *names):
    for name in names:
        assert [d for n, d in calls if n == name] == [torch.device("meta")], name


def test_feed_forward(asked):
    from fovi_b200 import ops
    leaves = [_meta(*s) for s in ((5, 16), (24, 16), (24, 16), (8, 24), (24,), (24,), (8,))]
    ops.gated_feed_forward(*leaves)
    _check(asked, "fovi_gated_ffn_workspace_bytes", "fovi_gated_ffn_forward")
    asked.clear()
    ops.gated_feed_forward_backward(*leaves[:4], _meta(64, dtype=torch.uint8), _meta(5, 8))
    _check(asked, "fovi_gated_ffn_workspace_bytes", "fovi_gated_ffn_backward")


def test_attention(asked):
    from fovi_b200 import ops
    q, k, v = _meta(2, 5, 4, 16), _meta(2, 7, 4, 16), _meta(2, 7, 4, 16)
    o, lse = ops.attention(q, k, v, want_lse=True)
    _check(asked, "fovi_attention_workspace_bytes", "fovi_attention_forward")
    asked.clear()
    ops.attention_backward(q, k, v, o, _meta(2, 5, 4, 16), lse)
    _check(asked, "fovi_attention_workspace_bytes", "fovi_attention_backward")
