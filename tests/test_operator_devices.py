"""CPU: the device that is current when an entry point of the library is called, from the autograd Functions of the operators.  A default
stream's handle names no device, so tensors on another device than the caller's current one must bring theirs along."""
from types import SimpleNamespace

import pytest
import torch

from aotriton_b200 import autograd, cabi


@pytest.fixture
def calls(monkeypatch):
    """(entry point, current device) of each call; the entry points do nothing."""
    current, seen = [None], []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            current.append(self.device)

        def __exit__(self, *exc):
            current.pop()

    def entry(name, result=0):
        def call(*args, **kw):
            seen.append((name, current[-1]))
            return result
        return call

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=0))
    for name, result in (("sink_attn_fwd", 0), ("sink_attn_bwd", 0), ("sink_attn_bwd_workspace", 8), ("dropout", 0)):
        monkeypatch.setattr(cabi, name, entry(name, result))
    names = [("ab200_relative_bias_fwd", 0), ("ab200_relative_bias_bwd", 0), ("ab200_relative_bias_workspace", 8)]
    monkeypatch.setattr(cabi, "lib", lambda: SimpleNamespace(**{name: entry(name, result) for name, result in names}))
    monkeypatch.setattr(autograd._native, "note_bwd_family", lambda: None)
    return seen


HERE = torch.device("cpu")


def test_sink_attention(calls):
    q, k, v = (torch.zeros(1, 2, 5, 8, requires_grad=True) for _ in range(3))
    autograd._SinkAttention.apply(q, k, v, None, None, 0, 0, 3, 1, 1.0, False, 0).sum().backward()
    assert calls == [(name, HERE) for name in ("sink_attn_fwd", "sink_attn_bwd_workspace", "sink_attn_bwd")]


def test_relative_bias(calls):
    table = torch.zeros(8, 2, requires_grad=True)
    autograd._RelativeBias.apply(table, 5, 6, 2, (1, 2, 3), True, 0, torch.float32).sum().backward()
    assert calls == [(f"ab200_relative_bias_{name}", HERE) for name in ("fwd", "workspace", "bwd")]


def test_dropout(calls):
    x, r = (torch.zeros(3, 4, requires_grad=True) for _ in range(2))
    autograd._Dropout.apply(x, r, 0.5, 1, 2).sum().backward()
    assert calls == [("dropout", HERE)] * 2
