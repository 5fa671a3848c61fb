"""Sink attention in 64 bits with a bound of what the kernels' arithmetic may be off by, element for element.

Counted are the roundings: scores, sums and exponentials in fp32 (together `slop` of a probability: D + 4 additions and products of the
score at 2^-24 of the sum of its terms' magnitudes, as many again for the exponent's reference point, 2^-20 for the exponential and the sum), P and dS rounded to the type before the products
(eps / 2 each; fp16 values below its normal range 2^-25), O rounded where delta = rowsum(O dO) reads it, and the results (eps / 2).  fp32 sums over n keys or queries: n * 2^-24 of their terms' magnitudes.
"""
from __future__ import annotations

import torch

from oracle import attention as A
from oracle import layer as O


def reference(q, k, v, window, sinks, sm_scale, dout=None):
    """One sequence batch (dense): (values, bounds), dicts over out, lse and, with dout, dq, dk, dv.  CPU or GPU, all in 64 bits."""
    dt = q.dtype
    half, tiny = torch.finfo(dt).eps / 2 * 1.001, 2.0 ** -25 if dt == torch.float16 else 0.0
    b, hq, sq, d = q.shape
    g = hq // k.shape[1]
    sk = k.shape[2]
    mask = O.sink_mask(sq, sk, window, sinks).to(q.device)
    Q, K, V = q.double(), k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    r = A.attention(q, k, v, sm_scale=sm_scale, mask=mask, dout=dout, acc_dtype=torch.float64)
    s = (Q @ K.transpose(-1, -2)) * sm_scale
    p = torch.where(mask, torch.exp(s - torch.where(torch.isinf(r.lse), 0.0, r.lse)[..., None]), 0.0)
    size = (Q.abs() @ K.abs().transpose(-1, -2)) * abs(sm_scale)
    slop = 2 * (d + 4) * 2.0 ** -24 * float(torch.where(mask, size, 0.0).max() if mask.any() else 0) + 2.0 ** -20 + max(sq, sk) * 2.0 ** -24
    out = p @ V
    values = dict(out=out, lse=r.lse)
    seen = mask.double()
    e_out = (half + slop) * (p @ V.abs()) + tiny * (seen @ V.abs()) + half * out.abs()
    bounds = dict(out=e_out, lse=torch.full_like(r.lse, 0.0) + slop * 2 + 2.0 ** -22 * torch.where(torch.isinf(r.lse), 0.0, r.lse).abs() + 1e-6)
    if dout is None:
        return values, bounds
    D = dout.double()
    fold = lambda t: t.view(b, hq // g, g, *t.shape[2:]).sum(2)
    dp = D @ V.transpose(-1, -2)
    delta = (out * D).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dp_size = D.abs() @ V.abs().transpose(-1, -2)
    e_delta = (e_out * D.abs()).sum(-1, keepdim=True) + d * 2.0 ** -24 * (out.abs() * D.abs()).sum(-1, keepdim=True)
    e_ds = half * ds.abs() + slop * p * (dp_size + delta.abs()) + p * e_delta + tiny * seen
    e_p = (half + slop) * p + tiny * seen
    T = lambda t: t.transpose(-1, -2)
    values.update(dq=ds @ K * sm_scale, dk=fold(T(ds) @ Q) * sm_scale, dv=fold(T(p) @ D))
    n = g * sq
    more = lambda a, x: n * 2.0 ** -24 * fold(T(a) @ x)
    bounds.update(dq=e_ds @ K.abs() * sm_scale + sk * 2.0 ** -24 * (ds.abs() @ K.abs()) * sm_scale,
                  dk=(fold(T(e_ds) @ Q.abs()) + more(ds.abs(), Q.abs())) * sm_scale, dv=fold(T(e_p) @ D.abs()) + more(p, D.abs()))
    for name in ("dq", "dk", "dv"):
        bounds[name] = bounds[name] + half * values[name].abs() + (2.0 ** -25 if dt == torch.float16 else 1e-37)
    return values, bounds


def check(name, got, values, bounds):
    want, bound = values[name], bounds[name]
    got = got.double().reshape(want.shape)
    assert not torch.isnan(got).any(), f"{name}: NaN"
    infinite = torch.isinf(want)
    assert torch.equal(got[infinite], want[infinite]), name
    off = (got - want).abs()[~infinite] - bound[~infinite]
    assert not off.numel() or float(off.max()) <= 0, f"{name}: beyond its bound by {float(off.max()):.3g}"
