"""GPU: the operators over a paged cache and latent attention where a call is not the ordinary one: waits that run out, the Python way, compiled callers, other
modes, captured training steps."""
import pytest
import torch

from _paged_reference import make
from aotriton_b200 import autograd, cabi, paged

pytestmark = pytest.mark.gpu


def _paged_call(kind):
    """(run, status range of its kernel)."""
    if kind == "paged":
        q, kc, vc, table, lens = make(3, 8, 2, 1, 128, 128, 16, [900, 40, 300], torch.bfloat16)
        return lambda: paged.paged_attention(q, kc, vc, table, lens), (0x6000, 0x7000)
    if kind == "rows":
        q, kc, vc, table, lens = make(2, 32, 2, 2, 64, 64, 32, [900, 40], torch.float16)
        return lambda: paged.paged_attention(q, kc, vc, table, lens), (0x6000, 0x7000)
    heads, sq = {"latent16": (16, 1), "latent32": (32, 1), "latent64": (128, 1), "latent_queries": (16, 3)}[kind]
    q, cache, _, table, lens = make(3, heads, 1, sq, 576, 512, 64, [900, 40, 300], torch.bfloat16, shared=True)
    return lambda: paged.paged_latent_attention(q, cache[:, :, 0], table, lens, 512, 0.07), (0x7000, 0x8000)


KINDS = ["paged", "rows", "latent16", "latent32", "latent64", "latent_queries"]


@pytest.mark.parametrize("kind", KINDS)
def test_waits_run_out_cleanly(kind):
    """One copy is left out with a wait limit of about a million cycles: the kernel returns, the status word names it, further work is refused until the
    reset, and the next call gives what an undisturbed one gives."""
    L = cabi.lib()
    call, (lo, hi) = _paged_call(kind)
    stream = torch.cuda.current_stream().cuda_stream
    assert L.ab200_kernel_status(1) == 0
    want = call()
    torch.cuda.synchronize()
    L.ab200_debug_bounded_wait_test(1, 1000)
    try:
        call()
        call()      # queued behind the first: starts after the failure and leaves at once
    finally:
        L.ab200_debug_bounded_wait_test(0, 0)
    assert L.ab200_stream_check(stream) == 719
    code = L.ab200_kernel_status(0)
    assert lo <= code < hi, hex(code)
    with pytest.raises(RuntimeError, match="hipErrorLaunchFailure"):
        call()
    assert L.ab200_kernel_status(1) == code
    assert L.ab200_stream_check(stream) == 0
    assert torch.equal(call(), want)


@pytest.mark.parametrize("kind", KINDS)
def test_the_python_way(kind, monkeypatch):
    call, _ = _paged_call(kind)
    want = call()
    monkeypatch.setattr(paged._native, "paged_attention", lambda *a: None)
    assert torch.equal(call(), want)


def test_the_python_way_of_the_books(monkeypatch):
    def run():
        table = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
        n, m = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 0, 0], [40, 0, 100]))
        r = paged.block_tables(table, n, m, torch.arange(30, dtype=torch.int32, device="cuda").flip(0).contiguous(), 16, 150)
        cache = torch.zeros(30, 16, 2, 24, device="cuda", dtype=torch.float16)
        x = torch.arange(150 * 2 * 24, device="cuda").view(150, 2, 24).half()
        paged.paged_write(x, None, cache, None, r.slots)
        return table, *r, cache

    want = run()
    for name in ("block_tables", "paged_write"):
        monkeypatch.setattr(paged._native, name, lambda *a: None)
    for a, b in zip(run(), want):
        assert torch.equal(a, b)


def test_compiled_callers():
    call, _ = _paged_call("paged")
    torch._dynamo.reset()
    assert torch.equal(torch.compile(lambda: call() * 2, backend="eager")(), call() * 2)
    table = torch.full((2, 5), -1, dtype=torch.int32, device="cuda")
    n, m, free = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 3], [5, 30], [4, 3, 2, 1, 0]))
    cache = torch.zeros(5, 16, 1, 8, device="cuda")
    x = torch.randn(35, 1, 8, device="cuda")

    def step():
        r = paged.block_tables(table, n, m, free, 16, 35)
        paged.paged_write(x, None, cache, None, r.slots)
        return r.slots + 1

    torch._dynamo.reset()
    slots = torch.compile(step, backend="eager")() - 1
    assert table[:, :3].tolist() == [[4, -1, -1], [-1, 3, 2]] and torch.equal(slots, paged.block_tables(table, n, m, free, 16, 35).slots)
    assert torch.equal(cache.view(80, 8)[slots[:5]], x[:5, 0])
    q, k, r, v = (torch.randn(1, h, 20, d, device="cuda").half().requires_grad_() for h, d in ((2, 96), (2, 64), (1, 32), (2, 64)))
    want = autograd.latent_attention(q, k, r, v, causal=True)
    torch._dynamo.reset()
    got = torch.compile(lambda: autograd.latent_attention(q, k, r, v, causal=True) * 2, backend="eager")()
    assert torch.equal(got, want * 2)
    for a, b in zip(torch.autograd.grad(got.sum(), (q, k, r, v)), torch.autograd.grad(want.sum() * 2, (q, k, r, v))):
        assert torch.equal(a, b)


def test_forward_mode_and_transforms_are_refused():
    import torch.autograd.forward_ad as fwd
    q, kc, vc, table, lens = make(2, 8, 2, 1, 64, 64, 16, [90, 40], torch.float16)
    with fwd.dual_level(), pytest.raises(RuntimeError):
        paged.paged_attention(fwd.make_dual(q, torch.ones_like(q)), kc, vc, table, lens)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: paged.paged_attention(t, kc, vc, table, lens).float().sum())(q)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: paged.paged_attention(t, kc, vc, table, lens))(torch.stack([q, q]))


def _inputs(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(2, h, 100, d, generator=g, device="cuda").half().requires_grad_() for h, d in ((4, 192), (2, 128), (1, 64), (2, 128))]


@pytest.mark.parametrize("packed", [False, True])
def test_latent_attention_the_python_way(packed, monkeypatch):
    ins = _inputs()
    if packed:
        ins = [t.detach()[:1].requires_grad_() for t in ins]
        ends = torch.tensor([0, 30, 90], dtype=torch.int32, device="cuda")      # (ten rows behind the last sequence)
        call = lambda: autograd.varlen_latent_attention(*ins, ends, ends, 60, 60, causal=True, return_lse=True)
    else:
        call = lambda: autograd.latent_attention(*ins, causal=True, return_lse=True)
    out, lse = call()
    do = torch.randn_like(out)
    want = torch.autograd.grad(out, ins, do)
    monkeypatch.setattr(autograd._native, "latent_attend", lambda *a: None)
    again, lse2 = call()
    assert torch.equal(again, out) and (packed or torch.equal(lse, lse2))
    for a, b in zip(torch.autograd.grad(again, ins, do), want):
        assert torch.equal(a, b)
    if packed:
        assert (out[:, :, 90:] == 0).all() and all((g[:, :, 90:] == 0).all() for g in want)


@pytest.mark.parametrize("native", [True, False])
def test_hooks_modes_and_second_derivatives(native, monkeypatch):
    if not native:
        monkeypatch.setattr(autograd._native, "latent_attend", lambda *a: None)
    ins = _inputs()
    call = lambda: autograd.latent_attention(*ins, causal=True)
    out = call()
    do = torch.randn_like(out)
    want = torch.autograd.grad(out, ins, do)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        out = call()
    for a, b in zip(torch.autograd.grad(out, ins, do), want):
        assert torch.equal(a, b)
    for change in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t[..., : t.shape[-1] // 2], lambda t: t.flatten()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            out = call()
        with pytest.raises(ValueError, match="came back"):
            torch.autograd.grad(out, ins, do)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(call(), ins, torch.stack([do] * 2), is_grads_batched=True)
    grads = torch.autograd.grad(call(), ins, do.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(grads[0].float().sum(), ins[0])
    turned = torch.randn(2, 4, 128, 100, device="cuda").half().transpose(2, 3)      # a gradient without unit stride
    for a, b in zip(torch.autograd.grad(call(), ins, turned), torch.autograd.grad(call(), ins, turned.contiguous())):
        assert torch.equal(a, b)


def test_a_captured_training_step_beside_an_eager_graph():
    ins = _inputs()
    keep = autograd.latent_attention(*ins, causal=True)      # an eager graph of the same leaves, alive throughout
    do = torch.randn_like(keep)
    want = torch.autograd.grad(autograd.latent_attention(*ins, causal=True), ins, do)
    detached = [t.detach().requires_grad_() for t in ins]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(autograd.latent_attention(*detached, causal=True), detached, do)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = autograd.latent_attention(*detached, causal=True)
        grads = torch.autograd.grad(out, detached, do)
    for t in (out, *grads):
        t.detach().zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, keep)
    for a, b in zip(grads, want):
        assert torch.equal(a, b)
    for a, b in zip(torch.autograd.grad(keep, ins, do), want):
        assert torch.equal(a, b)


def test_gradients_of_some_inputs_alone():
    ins = _inputs()
    out = autograd.latent_attention(*ins)
    do = torch.randn_like(out)
    want = torch.autograd.grad(out, ins, do)
    for i in range(4):
        some = [t if j == i else t.detach() for j, t in enumerate(ins)]
        (got,) = torch.autograd.grad(autograd.latent_attention(*some), some[i], do)
        assert torch.equal(got, want[i])
    with torch.no_grad():
        assert torch.equal(autograd.latent_attention(*ins), out)
    o, lse = autograd.latent_attention(*ins, return_lse=True)
    assert torch.equal(o, out) and lse.shape == (8, 100)
