"""Calls from compiled code: the graph breaks at the Functions, whose results and gradients are the uncompiled call's."""
import pytest
import torch

from test_gpu_layer_modes import CALLS, _healthy, _rand

pytestmark = pytest.mark.gpu


def _attention(ins, **kw):
    from aotriton_b200 import autograd
    return autograd.attention(*ins, causal=True, **kw)


def _varlen_attention(ins):
    from aotriton_b200 import autograd
    ends = torch.tensor([0, 30, 100], dtype=torch.int32, device="cuda")
    return autograd.varlen_attention(*ins, ends, ends, 70, 70)


_QKV = CALLS["sink"][1]
CALLS = CALLS | {"attention": (_attention, _QKV), "attention_dropout": (lambda ins: _attention(ins, dropout_p=0.2), _QKV), "varlen_attention": (_varlen_attention, _QKV)}


@pytest.mark.parametrize("kind", list(CALLS))
def test_a_compiled_caller(kind):
    call, inputs = CALLS[kind]
    ins = inputs()
    do = torch.randn_like(call(ins))
    want_out = call(ins)
    want = torch.autograd.grad(want_out, ins, do)
    torch._dynamo.reset()
    out = torch.compile(lambda a: call(a) * 2, backend="eager")(ins)
    assert torch.equal(out, want_out * 2)
    for a, b in zip(torch.autograd.grad(out, ins, do / 2), want):
        assert torch.equal(a, b)
    _healthy()


def test_a_compiled_layer_step():
    """Bias, attention and dropout with the residual in one compiled function, with gradients."""
    from aotriton_b200 import autograd
    q, k, v, r = (_rand(1, 4, 48, 64, seed=i) for i in range(4))
    table = _rand(32, 4, seed=5)
    ins = (q, k, v, r, table)

    def layer():
        bias = autograd.relative_position_bias(table, 48, 48)
        return autograd.dropout(autograd.attention(q, k, v, bias, dropout_p=0.1), 0.1, residual=r) + 1

    torch._dynamo.reset()
    compiled = torch.compile(layer, backend="eager")
    do = torch.randn_like(q)
    want, got = layer(), compiled()
    assert torch.equal(want, got)
    for a, b in zip(torch.autograd.grad(got, ins, do), torch.autograd.grad(want, ins, do)):
        assert torch.equal(a, b)
    _healthy()
