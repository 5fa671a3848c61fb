"""Sink attention with head dims of one: a single column may have any stride, which contiguous() leaves as it is."""
import pytest
import torch

from _sink_reference import check, reference

pytestmark = pytest.mark.gpu


def _spread(t):
    """t's values, the innermost axis the slowest in memory."""
    return t.transpose(2, 3).clone(memory_format=torch.contiguous_format).transpose(2, 3)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,Dv", [(1, 1), (1, 5), (3, 1), (1, 64), (64, 1)])
@pytest.mark.parametrize("Sq", [1, 5, 70])
@pytest.mark.parametrize("operands", ["as they come", "spread", "gradient spread"])
def test_one_column(operands, Sq, D, Dv, dt):
    from aotriton_b200 import autograd
    g = torch.Generator(device="cuda").manual_seed(Sq + D)
    q, k, v, do = (torch.randn(1, h, s, d, generator=g, device="cuda").to(dt) for h, s, d in ((4, Sq, D), (2, 90, D), (2, 90, Dv), (4, Sq, Dv)))
    if operands == "spread":
        q, k, v = map(_spread, (q, k, v))
        assert D > 1 or k.stride(-1) == 90
    if operands != "as they come":
        do = _spread(do)
    for t in (q, k, v):
        t.requires_grad_()
    out, lse = autograd.sink_attention(q, k, v, 30, 4, return_lse=True)
    grads = torch.autograd.grad(out, (q, k, v), do)
    values, bounds = reference(q.detach(), k.detach(), v.detach(), 30, 4, D ** -0.5, do)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out.detach(), lse) + grads):
        check(name, got, values, bounds)
