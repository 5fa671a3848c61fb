"""GPU: the gradient of columns that all heads share is summed from 32 bits and rounded once, where the kernels leave 32-bit columns."""
import pytest
import torch

from aotriton_b200 import autograd, cabi

pytestmark = pytest.mark.gpu
KEYS = QUERIES = 256
SCALE = 0.125


def _whole_numbers(h, hk, dn, dr, dv, dtype, device):
    """Inputs for which all but the last rounding is exact, and the shared columns' gradient of each kv head, (hk, keys, dr), in whole multiples of SCALE / 256.

    Keys are zero: each of the 256 has the weight 2^-8 (a rounding to the type takes the exponential's last bits away).  Values are one in the first column for
    even keys and minus one for odd ones: the output is zero, dP = +-dO, dS = +-dO / 256 with dO = +-1.  So a head's share is a sum of 256 queries' whole numbers
    below 128 -- up to 15 bits, which 32 hold and 16 do not; every second kv head has the other sign but for the last query, so that their sum is small beside them."""
    g = torch.Generator().manual_seed(7)
    group = h // hk
    number = torch.randint(0, 128, (1, hk, QUERIES, dn + dr), generator=g).double()
    number[:, 1::2, :-1] = number[:, ::2, :-1]
    do = torch.zeros(1, hk, QUERIES, dv, dtype=torch.float64)
    do[..., 0] = torch.where(torch.rand(QUERIES, generator=g) < 0.3, -1.0, 1.0)
    do[:, 1::2] *= -1
    sign = torch.where(torch.arange(KEYS) % 2 == 0, 1.0, -1.0).double()
    share = sign[None, :, None] * (do[0, :, :, :1] * number[0, :, :, dn:]).sum(1, keepdim=True) * group
    q, do = (t.repeat_interleave(group, 1).to(device, dtype) for t in (number, do))
    k, r = torch.zeros(1, hk, KEYS, dn, device=device, dtype=dtype), torch.zeros(1, 1, KEYS, dr, device=device, dtype=dtype)
    v = torch.zeros(1, hk, KEYS, dv, device=device, dtype=dtype)
    v[..., 0] = sign.to(device, dtype)
    return (q, k, r, v), do, share


@pytest.mark.parametrize("h,hk", [(32, 32), (40, 40), (48, 24)])      # 16 heads at a time, and some more
@pytest.mark.parametrize("dn,dr,dv", [(128, 64, 128), (192, 64, 256), (64, 32, 64), (40, 24, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rounded_once(dtype, h, hk, dn, dr, dv):
    inputs, do, share = _whole_numbers(h, hk, dn, dr, dv, dtype, "cuda")
    want = (share.sum(0) * (SCALE / 256)).to(dtype)
    shares_rounded = ((share * (SCALE / 256)).to(dtype).double().sum(0)).to(dtype)
    assert (shares_rounded != want).double().mean() > 0.5      # (what the sum of rounded shares gives is another thing)
    q, k, r, v = (t.requires_grad_() for t in inputs)
    joined = torch.cat([k, r.expand(-1, hk, -1, -1)], -1).detach()
    lse = torch.empty(h, QUERIES, device="cuda")
    assert cabi.attn_bwd_shared_workspace(q, joined, v, do, do, q, joined, v, lse, lse, dr, sm_scale=SCALE) == hk * KEYS * dr
    out = autograd.latent_attention(q, k, r, v, sm_scale=SCALE)
    assert (out == 0).all()
    (got,) = torch.autograd.grad(out, r, do)
    assert torch.equal(got[0, 0].cpu(), want)


def _bounds(inputs, do, scale, dtype):
    """Output, gradients and what each may be off by, of one causal sequence: as in the entry's test, for all of them."""
    q, k, r, v = (t[0].double() for t in inputs)
    do, h, dn = do[0].double(), q.shape[0], k.shape[2]
    u, least = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0
    kk = torch.cat([k, r.expand(h, -1, -1)], -1)
    x = q @ kk.transpose(1, 2) * scale
    hidden = torch.ones(x.shape[-2:], dtype=torch.bool, device=x.device).triu(1)
    p = torch.softmax(x.masked_fill(hidden, -float("inf")), -1)
    o, dp = p @ v, do @ v.transpose(1, 2)
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    mixed, n = p @ v.abs(), x.shape[1]
    score = ((q.shape[2] + 8) * 2.0 ** -24 * scale * (q.abs() @ kk.abs().transpose(1, 2)) + (x.abs() + 8) * 2.0 ** -23).masked_fill(hidden, 0).amax(-1, keepdim=True)
    weight = 1.05 * u + 3 * score + n * 2.0 ** -24
    output = weight * mixed + u * 1.05 * o.abs() + least * (v.abs().sum(1, keepdim=True) + 1)
    terms = p * (do.abs() @ v.abs().transpose(1, 2) + (do.abs() * mixed).sum(-1, keepdim=True))
    off = 1.05 * u * ds.abs() + 1.05 * p * (do.abs() * output).sum(-1, keepdim=True) + (3 * score + (v.shape[2] + 8) * 2.0 ** -23) * terms + least
    sums = (n + h) * 2.0 ** -24
    dq, dk, dv = ds @ kk * scale, ds.transpose(1, 2) @ q * scale, p.transpose(1, 2) @ do
    most = [output, (off + sums * ds.abs()) @ kk.abs() * scale, (off + sums * ds.abs()).transpose(1, 2) @ q.abs() * scale,
            (weight * p + least).transpose(1, 2) @ do.abs()]
    want = [o, dq, dk[..., :dn], dk[..., dn:].sum(0, keepdim=True), dv]
    most = [most[0], most[1], most[2][..., :dn], most[2][..., dn:].sum(0, keepdim=True), most[3]]
    return want, [m + 1.05 * u * (w.abs() + m) + least for w, m in zip(want, most)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dn,dr,dv", [(128, 64, 128), (64, 32, 64)])
def test_packed_each_element_by_its_own_bound(dtype, dn, dr, dv):
    lens, h, scale = [5, 130, 1, 64], 4, (dn + dr) ** -0.5
    ends = torch.tensor([0, 5, 135, 136, 200], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, r, v, do = (torch.randn(1, 230, n, d, generator=g, device="cuda").to(dtype).transpose(1, 2) for n, d in ((h, dn + dr), (h, dn), (1, dr), (h, dv), (h, dv)))
    leaves = [t.detach().requires_grad_() for t in (q, k, r, v)]
    out = autograd.varlen_latent_attention(*leaves, ends, ends, 130, 130, causal=True)
    grads = torch.autograd.grad(out, leaves, do)
    at = 0
    for n in lens:
        part = [t[:, :, at:at + n].detach() for t in (q, k, r, v, do)]
        want, most = _bounds(part[:4], part[4], scale, dtype)
        for what, got, w, m in zip(("out", "dq", "dk", "dshared", "dv"), (out, *grads), want, most):
            assert ((got[0, :, at:at + n].double() - w).abs() <= m).all(), what
        at += n
    assert all((t[:, :, at:] == 0).all() for t in (out, *grads))
