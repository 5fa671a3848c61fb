"""CPU: the device that is current when an entry point of the library is called, from the autograd Functions of the operators.  A default
stream's handle names no device, so tensors on another device than the caller's current one must bring theirs along."""
from types import SimpleNamespace

import pytest
import torch

from aotriton_b200 import autograd, cabi, flash


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
    for name in ("attn_fwd", "attn_bwd", "attn_fwd_varlen", "attn_bwd_varlen"):
        monkeypatch.setattr(flash, name, entry(name))
    for name in ("eager_delta", "lazy_delta", "lazy_dq_acc"):
        monkeypatch.setattr(flash, name, lambda t: None)
    monkeypatch.setattr(autograd, "_check", lambda err, what: None)
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


def _qkv():
    return [torch.zeros(1, 2, 5, 8, requires_grad=True) for _ in range(3)]


@pytest.mark.parametrize("dropout_p", [0.0, 0.1])
def test_attention(calls, dropout_p):
    autograd._Attention.apply(*_qkv(), None, False, 1.0, dropout_p).sum().backward()
    ends = torch.tensor([0, 2, 5], dtype=torch.int32)
    autograd._VarlenAttention.apply(*_qkv(), ends, ends, 3, 3, False, 1.0, dropout_p).sum().backward()
    assert calls == [(name, HERE) for name in ("attn_fwd", "attn_bwd", "attn_fwd_varlen", "attn_bwd_varlen")]


def test_attention_operators(calls):
    autograd.op_attn_fwd(*_qkv(), None, 1.0, 0.0, 0, 0, 0, 1, 2)[0].sum().backward()
    assert calls == [(name, HERE) for name in ("attn_fwd", "attn_bwd")]
