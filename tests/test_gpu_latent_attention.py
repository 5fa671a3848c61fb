"""GPU: latent attention, absorbed over a paged cache and expanded with its gradients, against definitions in 64 bits."""
import math

import pytest
import torch

from _paged_reference import check, make, reference
from aotriton_b200 import autograd, cabi, paged

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]
ALL = HALF + [torch.float32]


def run(b, h, sq, d, dv, page, lengths, dtype, query_lengths=None, **kw):
    q, cache, _, table, lens = make(b, h, 1, sq, d, dv, page, lengths, dtype, shared=True, query_lengths=query_lengths, **kw)
    ql = None if query_lengths is None else torch.tensor(query_lengths, dtype=torch.int32, device="cuda")
    scale = (d // 3) ** -0.5
    out, lse = paged.paged_latent_attention(q, cache[:, :, 0], table, lens, dv, scale, query_lengths=ql, return_lse=True)
    want, want_lse, most = reference(q, cache, cache[..., :dv], table, lens, query_lengths=ql, sm_scale=scale)
    check(out, want, most)
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty)
    assert ((lse.double() - want_lse)[~empty].abs() < 1e-3).all()
    assert cabi.lib().ab200_kernel_status(0) == 0


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("h", [1, 5, 8, 16, 20, 32, 64, 100, 128])
def test_heads(dtype, h):
    run(3, h, 1, 576, 512, 64, [300, 1, 129], dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 8, 48, 1, 5])
def test_pages(dtype, page):
    lengths = [0, 1, page, page + 1, 127, 128, 129, 700]
    run(len(lengths), 16, 1, 576, 512, page, lengths, dtype, bad=1)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("d,dv", [(288, 256), (576, 576), (192, 128), (320, 256), (512, 512), (40, 24), (7, 5), (640, 512), (576, 64)])
def test_widths(dtype, d, dv):
    run(2, 12, 1, d, dv, 32, [200, 33], dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("sq", [2, 3, 9])
def test_several_queries(dtype, sq):
    run(5, 16, sq, 576, 512, 64, [2, 150, 64, 0, 400], dtype, query_lengths=[sq, 1, sq, sq, 0])
    run(2, 128, sq, 576, 512, 16, [260, 5], dtype)


@pytest.mark.parametrize("h", [16, 64, 128])
def test_long_and_ragged(h):
    run(1, h, 1, 576, 512, 64, [20001], torch.bfloat16)
    run(40, h, 1, 576, 512, 16, [(i * 37) % 300 + (3000 if i == 7 else 0) for i in range(40)], torch.float16)


@pytest.mark.parametrize("dtype,h", [(torch.bfloat16, 16), (torch.float16, 32), (torch.bfloat16, 64), (torch.float16, 100), (torch.float32, 4)])
def test_many_sequences(dtype, h):
    run(130, h, 1, 192, 128, 16, [(i * 53) % 200 + (900 if i in (3, 129) else 0) for i in range(130)], dtype)
    run(65, h, 2, 288, 256, 32, [(i * 53) % 100 for i in range(65)], dtype, query_lengths=[i % 3 for i in range(65)])


def test_many_rows_a_sequence():
    run(2, 128, 11, 192, 128, 16, [300, 40], torch.bfloat16)      # more chunks of rows than stand side by side


@pytest.mark.parametrize("dtype", HALF)
def test_weights_that_grow_along_the_sequence(dtype):
    # each tile's largest score is above the last one's: what has been summed is rescaled again and again
    q, cache, _, table, lens = make(1, 32, 1, 1, 576, 512, 64, [1000], dtype, shared=True, poison=False)
    q.fill_(0.0)
    q[..., 0] = 1.0
    pos = torch.arange(1000, device="cuda")
    cache[table[0, pos // 64].long(), pos % 64, 0, 0] = (pos.float() / 8).to(dtype)
    scale = 0.5
    out = paged.paged_latent_attention(q, cache[:, :, 0], table, lens, 512, scale)
    want, _, most = reference(q, cache, cache[..., :512], table, lens, sm_scale=scale)
    check(out, want, most)


def test_strides_and_captured_call():
    q, cache, _, table, lens = make(3, 16, 1, 1, 576, 512, 64, [100, 2000, 7], torch.bfloat16, shared=True)
    want = paged.paged_latent_attention(q, cache[:, :, 0], table, lens, 512, 0.07)
    wide = torch.full((*cache.shape[:2], 640), float("nan"), device="cuda", dtype=cache.dtype)
    wide[..., 64:].copy_(cache[:, :, 0])
    assert torch.equal(paged.paged_latent_attention(q, wide[..., 64:], table, lens, 512, 0.07), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(paged.paged_latent_attention(q, cache[:, :, 0], table, lens, 512, 0.07), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.paged_latent_attention(q, cache[:, :, 0], table, lens, 512, 0.07)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)


# ---- expanded ---------------------------------------------------------------------------------------------------
def _expanded(q, k, r, v, do, causal, scale):
    """Output, the four gradients, and what they may be off by, in 64 bits."""
    h, g = q.shape[1], q.shape[1] // k.shape[1]
    q, k, r, v, do = (t.double() for t in (q, k, r, v, do))
    kk = torch.cat([k, r.expand(-1, k.shape[1], -1, -1)], -1).repeat_interleave(g, 1)
    vv = v.repeat_interleave(g, 1)
    x = q @ kk.transpose(-1, -2) * scale
    if causal:
        x = x.masked_fill(torch.ones(x.shape[-2:], dtype=torch.bool, device=x.device).triu(1), -math.inf)
    p = torch.softmax(x, -1)
    out = p @ vv
    dp = do @ vv.transpose(-1, -2)
    ds = p * (dp - (do * out).sum(-1, keepdim=True)) * scale
    dk = (ds.transpose(-1, -2) @ q).unflatten(1, (-1, g)).sum(2)
    dv = (p.transpose(-1, -2) @ do).unflatten(1, (-1, g)).sum(2)
    dn = k.shape[-1]
    return out, ds @ kk, dk[..., :dn], dk[..., dn:].sum(1, keepdim=True), dv


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("b,h,hk,s,dn,dr,dv", [(1, 2, 2, 130, 128, 64, 128), (2, 4, 4, 77, 64, 32, 64), (1, 4, 2, 1, 96, 32, 80), (1, 3, 3, 50, 13, 3, 10),
                                               (1, 2, 2, 200, 192, 64, 256)])
@pytest.mark.parametrize("causal", [True, False])
def test_expanded_and_gradients(dtype, b, h, hk, s, dn, dr, dv, causal):
    g = torch.Generator(device="cuda").manual_seed(3)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    q = rand(b, s, h, dn + dr).transpose(1, 2).requires_grad_()
    kv = rand(b, s, hk, dn + dv).transpose(1, 2)
    k, v = kv[..., :dn].requires_grad_(), kv[..., dn:].requires_grad_()
    r = rand(b, 1, s, dr).requires_grad_()
    do = rand(b, h, s, dv)
    out = autograd.latent_attention(q, k, r, v, causal=causal)
    grads = torch.autograd.grad(out, (q, k, r, v), do)
    want = _expanded(q.detach(), k.detach(), r.detach(), v.detach(), do, causal, (dn + dr) ** -0.5)
    flat = {torch.bfloat16: 2e-2, torch.float16: 1e-2, torch.float32: 1e-4}[dtype]
    for got, w, what in zip((out, *grads), want, ("out", "dq", "dk", "dshared", "dv")):
        assert got.shape == w.shape and got.dtype == dtype
        # (the attention's flat tolerances; the shared columns' gradient is a sum over heads of such)
        n = h if what == "dshared" else 1
        assert ((got.double() - w).abs() <= flat * n * (1 + w.abs())).all(), (what, float((got.double() - w).abs().max()))


def test_shared_gradient_against_differences():
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, r, v = (torch.randn(1, n, 6, d, generator=g, device="cuda") for n, d in ((3, 12), (3, 8), (1, 4), (3, 5)))
    r.requires_grad_()
    c = torch.randn(1, 3, 6, 5, generator=g, device="cuda")
    (grad,) = torch.autograd.grad((autograd.latent_attention(q, k, r, v, causal=True) * c).sum(), r)
    step = 2.0 ** -6
    for i in range(6):
        for j in range(4):
            e = torch.zeros_like(r)
            e[0, 0, i, j] = step
            with torch.no_grad():
                up, down = ((autograd.latent_attention(q, k, r + s * e, v, causal=True).double() * c).sum() for s in (1, -1))
            # (third derivatives of a softmax over scores of order 1: below 10 step ** 2; rounding 2^-22 / step)
            assert abs(float((up - down) / (2 * step)) - float(grad[0, 0, i, j])) < 10 * step ** 2 + 1e-3


@pytest.mark.parametrize("dtype", HALF)
def test_packed(dtype):
    lens, h, dn, dr, dv = [5, 130, 1, 64], 4, 128, 64, 128
    ends = torch.tensor([0, 5, 135, 136, 200], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, r, v, do = (torch.randn(1, 200, n, d, generator=g, device="cuda").to(dtype).transpose(1, 2) for n, d in ((h, dn + dr), (h, dn), (1, dr), (h, dv), (h, dv)))
    leaves = [t.detach().requires_grad_() for t in (q, k, r, v)]
    out = autograd.varlen_latent_attention(*leaves, ends, ends, 130, 130, causal=True)
    grads = torch.autograd.grad(out, leaves, do)
    at = 0
    for n in lens:
        part = [t[:, :, at:at + n].detach() for t in (q, k, r, v, do)]
        want = _expanded(*part, True, (dn + dr) ** -0.5)
        flat = {torch.bfloat16: 2e-2, torch.float16: 1e-2}[dtype]
        for got, w in zip((out, *grads), want):
            assert ((got[:, :, at:at + n].double() - w).abs() <= flat * h * (1 + w.abs())).all()
        at += n


def test_expanded_and_absorbed_agree():
    """One token of a layer both ways, from a latent vector through a head's expansions."""
    g = torch.Generator(device="cuda").manual_seed(6)
    h, dn, dr, dv, lat, n = 16, 128, 64, 128, 512, 90

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float64)

    latent, rope, wk, wv = rand(n, lat), rand(n, dr), rand(h, lat, dn) * lat ** -0.5, rand(h, lat, dv) * lat ** -0.5
    qn, qr = rand(h, dn), rand(h, dr)
    half = torch.bfloat16
    k, v = torch.einsum("nl,hld->hnd", latent, wk), torch.einsum("nl,hld->hnd", latent, wv)
    q = torch.cat([qn, qr], -1)[None, :, None].to(half)
    expanded = autograd.latent_attention(q, k[None].to(half), rope[None, None].to(half), v[None].to(half))
    absorbed_q = torch.cat([torch.einsum("hd,hld->hl", qn, wk), qr], -1)[None, :, None].to(half)
    cache = torch.zeros(3, 32, lat + dr, device="cuda", dtype=half)
    paged.paged_write(latent.to(half)[:, None], rope.to(half)[:, None], cache[:, :, None, :lat], cache[:, :, None, lat:], torch.arange(n, device="cuda"))
    o = paged.paged_latent_attention(absorbed_q, cache, torch.arange(3, device="cuda", dtype=torch.int32)[None], torch.tensor([n], device="cuda", dtype=torch.int32),
                                     lat, (dn + dr) ** -0.5)
    absorbed = torch.einsum("bhsl,hld->bhsd", o.double(), wv)
    # inputs rounded to 8 bits on either way: scores of order 10 off by 2^-8 each product's share, values of order 1
    assert (expanded.double() - absorbed).abs().max() < 0.1
