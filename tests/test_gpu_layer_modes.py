"""The operators around attention where a pass is not the ordinary one: a batch of gradients, a mode around the backward alone, saved-tensor hooks,
forward-mode gradients, function transforms."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu
F16 = torch.float16


def _rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(F16).requires_grad_()


def _sink(ins):
    from aotriton_b200 import autograd
    return autograd.sink_attention(*ins, 30, 4)


def _packed(ins):
    from aotriton_b200 import autograd
    ends = torch.tensor([0, 30, 100], dtype=torch.int32, device="cuda")
    return autograd.varlen_sink_attention(*ins, ends, ends, 70, 70, 30, 4)


def _bias(ins):
    from aotriton_b200 import autograd
    return autograd.relative_position_bias(*ins, 40, 50, batch=2)


def _dropout(ins):
    from aotriton_b200 import autograd
    return autograd.dropout(ins[0], 0.3, residual=ins[1])


CALLS = {"sink": (_sink, lambda: [_rand(1, 2, 100, 64, seed=i) for i in range(3)]), "packed": (_packed, lambda: [_rand(1, 2, 100, 64, seed=i) for i in range(3)]),
         "bias": (_bias, lambda: [_rand(32, 4, seed=1)]), "dropout": (_dropout, lambda: [_rand(20, 33, seed=i) for i in range(2)])}
calls = pytest.mark.parametrize("kind", list(CALLS))


def _healthy():
    from aotriton_b200 import cabi
    torch.cuda.synchronize()
    assert cabi.lib().ab200_kernel_status(0) == 0


@calls
def test_a_batch_of_gradients(kind):
    """No rule for it: refused, and the graph is good for ordinary ones afterwards."""
    call, inputs = CALLS[kind]
    ins = inputs()
    out = call(ins)
    do = torch.randn(3, *out.shape, device="cuda").to(F16)
    want = torch.autograd.grad(call(ins), ins, do[0])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, ins, do, is_grads_batched=True, retain_graph=True)
    for a, w in zip(torch.autograd.grad(out, ins, do[0]), want):
        assert torch.equal(a, w)
    _healthy()


class _Names(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


@calls
def test_a_mode_around_the_backward_alone(kind):
    call, inputs = CALLS[kind]
    ins = inputs()
    do = torch.randn_like(call(ins))
    want = torch.autograd.grad(call(ins), ins, do)
    out = call(ins)
    mode = _Names()
    mode.seen = []
    with mode:
        got = torch.autograd.grad(out, ins, do)
    assert any("aten.empty" in s for s in mode.seen)      # the Function's gradients
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    _healthy()


@calls
def test_saved_tensor_hooks(kind):
    call, inputs = CALLS[kind]
    ins = inputs()
    do = torch.randn_like(call(ins))
    want = torch.autograd.grad(call(ins), ins, do)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        out = call(ins)
    for a, b in zip(torch.autograd.grad(out, ins, do), want):
        assert torch.equal(a, b)
    if kind in ("sink", "packed"):
        for change in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t[..., : t.shape[-1] // 2], lambda t: t.flatten()):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
                out = call(ins)
            with pytest.raises(ValueError, match="came back"):
                torch.autograd.grad(out, ins, do)
    _healthy()


def test_a_hook_that_shortens_the_values():
    """Rows of V fewer than those of K, everything else as it was."""
    from aotriton_b200 import autograd
    q, k = (_rand(1, 2, n, 64, seed=n) for n in (40, 90))
    v = _rand(1, 2, 90, 32, seed=3)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:, :, :50] if t.shape == v.shape else t):
        out = autograd.sink_attention(q, k, v, 30, 4)
    with pytest.raises(ValueError, match="came back"):
        out.sum().backward()


def test_seed_tensors_through_hooks():
    from aotriton_b200 import autograd
    x = _rand(20, 32, seed=1)
    seed, offset = (torch.tensor([n], device="cuda") for n in (5, 6))
    call = lambda: autograd.dropout(x, 0.3, philox_seed=seed, philox_offset=offset)
    want = torch.autograd.grad(call().sum(), x)[0]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        out = call()
    assert torch.equal(torch.autograd.grad(out.sum(), x)[0], want)
    for change in (lambda t: t.cpu(), lambda t: t.int()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            out = call()
        with pytest.raises(ValueError, match="philox"):
            out.sum().backward()


@calls
def test_forward_mode_and_transforms_are_refused(kind):
    import torch.autograd.forward_ad as fwd
    call, inputs = CALLS[kind]
    ins = inputs()
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        call([fwd.make_dual(t.detach(), torch.ones_like(t)) for t in ins])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: call([t] + ins[1:]).float().sum())(ins[0].detach())
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: call([t] + [x.detach() for x in ins[1:]]))(torch.stack([ins[0].detach()] * 2))
    _healthy()
