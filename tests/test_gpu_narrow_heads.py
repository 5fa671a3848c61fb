"""GPU: head dims 129 to 192 with values of up to 128, whose kernels have two query tiles a CTA (where there are enough of them) and dK and dV in one launch."""
import math

import pytest
import torch

from aotriton_b200 import autograd, cabi

pytestmark = pytest.mark.gpu
FLAT = {torch.bfloat16: 2e-2, torch.float16: 1e-2}      # (the attention's flat tolerances)


def _reference(q, k, v, do, seen):
    g = q.shape[1] // k.shape[1]
    q, k, v, do = (t.double() for t in (q, k, v, do))
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    scale = q.shape[-1] ** -0.5
    x = (q @ kk.transpose(-1, -2) * scale).masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e300)
    e = torch.exp(x - top)
    s = e.sum(-1, keepdim=True)
    p = e / torch.where(s > 0, s, 1)
    out = p @ vv
    ds = p * (do @ vv.transpose(-1, -2) - (do * out).sum(-1, keepdim=True)) * scale
    return out, ds @ kk, (ds.transpose(-1, -2) @ q).unflatten(1, (-1, g)).sum(2), (p.transpose(-1, -2) @ do).unflatten(1, (-1, g)).sum(2)


def _check(got, want, dtype, group):
    for a, b, n in zip(got, want, (1, 1, group, group)):      # (a key's gradients are sums over its group's heads)
        assert ((a.double() - b).abs() <= FLAT[dtype] * n * (1 + b.abs())).all(), float((a.double() - b).abs().max())


def _rand(*shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", list(FLAT))
@pytest.mark.parametrize("b,h,hk,sq,sk,dq,dv,causal", [(1, 16, 16, 1300, 1300, 192, 128, True), (2, 16, 4, 640, 640, 192, 128, False), (3, 8, 2, 900, 300, 136, 64, True),
                                                       (1, 4, 2, 130, 333, 160, 96, False), (2, 24, 24, 512, 512, 192, 128, (100, 0)), (1, 2, 1, 300, 1, 176, 8, False),
                                                       (1, 40, 8, 513, 257, 184, 120, (30, 40)), (1, 3, 3, 1, 129, 192, 128, False)])
def test_dense(dtype, b, h, hk, sq, sk, dq, dv, causal):
    q, k, v = (_rand(b, n, s, d, dtype=dtype, seed=i).requires_grad_() for i, (n, s, d) in enumerate(((h, sq, dq), (hk, sk, dq), (hk, sk, dv))))
    do = _rand(b, h, sq, dv, dtype=dtype, seed=9)
    out = autograd.attention(q, k, v, causal=causal)
    grads = torch.autograd.grad(out, (q, k, v), do)
    m, n = torch.arange(sq, device="cuda")[:, None], torch.arange(sk, device="cuda")[None]
    left, right = (sq, 0) if causal is True else causal if causal else (sq, sk)
    seen = (n >= m - left) & (n <= m + right)
    _check((out, *grads), _reference(q.detach(), k.detach(), v.detach(), do, seen), dtype, h // hk)
    assert cabi.lib().ab200_last_fwd_family() == 2 and autograd.last_bwd_family == 2 and cabi.lib().ab200_kernel_status(0) == 0


@pytest.mark.parametrize("dtype", list(FLAT))
def test_packed_with_nan_around(dtype):
    lens, h, hk = [5, 700, 1, 0, 333], 12, 4
    ends = torch.tensor([0, 5, 705, 706, 706, 1039], dtype=torch.int32, device="cuda")
    q, k, v = (_rand(1, 1100, n, d, dtype=dtype, seed=i) for i, (n, d) in enumerate(((h, 192), (hk, 192), (hk, 128))))
    for t in (q, k, v):
        t[:, 1039:] = float("nan")
    q, k, v = (t.transpose(1, 2).requires_grad_() for t in (q, k, v))
    out = autograd.varlen_attention(q, k, v, ends, ends, 700, 700, causal=True)
    do = _rand(1, 1100, h, 128, dtype=dtype, seed=9).transpose(1, 2)
    grads = torch.autograd.grad(out, (q, k, v), do)
    at = 0
    for n in lens:
        part = [t.detach()[:, :, at:at + n] for t in (q, k, v, do)]
        seen = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        if n:
            _check([t[:, :, at:at + n] for t in (out, *grads)], _reference(*part, seen), dtype, h // hk)
        at += n


@pytest.mark.parametrize("what,drop,lo,hi", [("forward", 1, 0x100, 0x1000), ("dK and dV", 2, 0x3000, 0x4000), ("dQ", 3, 0x3000, 0x4000)])
def test_waits_run_out_cleanly(what, drop, lo, hi):
    """As in the tests of the other kernels: one copy is left out with a wait limit of about a million cycles."""
    L = cabi.lib()
    q, k, v = (_rand(1, 16, 1300, d, dtype=torch.float16, seed=i) for i, d in enumerate((192, 192, 128)))
    do, out, lse, delta = torch.randn_like(v), torch.empty_like(v), *(torch.empty(16, 1300, device="cuda") for _ in range(2))
    grads = [torch.empty_like(t) for t in (q, k, v)]

    def call():
        if what == "forward":
            return cabi.attn_fwd(q, k, v, out, lse, sm_scale=0.07)
        return cabi.attn_bwd(q, k, v, out, do, *grads, lse, delta, sm_scale=0.07)

    stream = torch.cuda.current_stream().cuda_stream
    assert L.ab200_kernel_status(1) == 0
    assert cabi.attn_fwd(q, k, v, out, lse, sm_scale=0.07) == 0
    results = [out, lse] if what == "forward" else grads
    assert call() == 0
    torch.cuda.synchronize()
    want = [t.clone() for t in results]
    L.ab200_debug_bounded_wait_test(drop, 1000)
    try:
        assert call() == 0
        assert call() == 0
    finally:
        L.ab200_debug_bounded_wait_test(0, 0)
    assert L.ab200_stream_check(stream) == 719
    code = L.ab200_kernel_status(0)
    assert lo <= code < hi, hex(code)
    assert call() == 719 and L.ab200_kernel_status(1) == code and L.ab200_stream_check(stream) == 0
    for t in results:
        t.fill_(float("nan"))
    assert call() == 0
    torch.cuda.synchronize()
    for a, b in zip(results, want):
        assert torch.equal(a, b)
