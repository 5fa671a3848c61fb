"""CPU: saved-tensor hooks that hand back tensors of another type, size or device.  The backward refuses them before anything is launched."""
import pytest
import torch

from aotriton_b200 import autograd
from test_operator_devices import calls      # noqa: F401 (a fixture)


def _hooks(change):
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t, change)


def _named(name, change):
    """change() of the saved tensor of that many elements."""
    return lambda t: change(t) if t.numel() == name else t


def _sink(change, varlen=0):
    q = torch.zeros(1, 4, 7, 16, dtype=torch.float16, requires_grad=True)                              # 448 elements, as the output
    k, v = (torch.zeros(1, 2, n, 16, dtype=torch.float16, requires_grad=True) for n in (9, 9))         # 288
    ends = [torch.tensor([0, 3, n], dtype=torch.int32) if varlen else None for n in (7, 9)]            # 3
    with _hooks(change):
        return autograd._SinkAttention.apply(q, k, v, *ends, 7 if varlen else 0, 9 if varlen else 0, 3, 1, 1.0, False, varlen)


@pytest.mark.parametrize("which", [448, 288, 28])
@pytest.mark.parametrize("change", [lambda t: t.double(), lambda t: t.bfloat16(), lambda t: t[..., :3], lambda t: torch.cat([t, t, t], 1), lambda t: t.flatten(),
                                    lambda t: t.to("meta")], ids=["double", "bf16", "narrow", "more_heads", "flat", "device"])
def test_sink_attention(calls, which, change):      # noqa: F811
    out = _sink(_named(which, change))
    calls.clear()
    with pytest.raises(ValueError, match="came back"):
        out.sum().backward()
    assert not calls


@pytest.mark.parametrize("change", [lambda t: t.long(), lambda t: t.to("meta"), lambda t: t[:2].clone() if t[-1] == 9 else t])
def test_packed_sink_attention(calls, change):      # noqa: F811
    out = _sink(_named(3, change), varlen=1)
    calls.clear()
    with pytest.raises(ValueError, match="came back"):
        out.sum().backward()
    assert not calls


@pytest.mark.parametrize("change", [lambda t: t.int(), lambda t: t.float(), lambda t: t.to("meta"), lambda t: t.expand(2)])
def test_dropout(calls, change):      # noqa: F811
    x = torch.zeros(5, 8, requires_grad=True)
    seed, offset = (torch.tensor([n], dtype=torch.int64) for n in (1, 2))
    with _hooks(change):
        out = autograd._Dropout.apply(x, None, 0.5, seed, offset)
    calls.clear()
    with pytest.raises(ValueError, match="philox"):
        out.sum().backward()
    assert not calls


def test_what_comes_back_as_it_was(calls):      # noqa: F811
    for varlen in (0, 1):
        _sink(lambda t: t.clone(), varlen).sum().backward()
    x = torch.zeros(5, 8, requires_grad=True)
    with _hooks(lambda t: t.clone()):
        autograd._Dropout.apply(x, None, 0.5, torch.tensor([1]), torch.tensor([2])).sum().backward()
    assert [name for name, _ in calls].count("sink_attn_bwd") == 2 and [name for name, _ in calls].count("dropout") == 2
