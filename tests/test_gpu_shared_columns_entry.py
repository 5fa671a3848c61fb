"""GPU: the C entry of the backward for joined keys over packed, strided and padded batches, with a workspace and gradients that hold NaN beforehand: what a C
caller may rely on, nothing cleared for the entry."""
import math

import pytest
import torch

from aotriton_b200 import cabi

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]
# keys of a sequence (none, fewer and more than queries), its queries
LENGTHS = [(7, 5), (130, 130), (0, 3), (40, 0), (64, 64), (200, 131), (0, 0), (1, 2)]
MAX_K, MAX_Q = 200, 131
# head dims of all kernels that leave 32-bit columns (one launch for dK and dV, wide heads, 128 and 64 columns), and of the general ones, which leave none
DIMS = [(128, 64, 128, True), (192, 64, 256, True), (64, 32, 64, True), (40, 24, 64, True), (13, 3, 10, False)]


def _places(layout):
    """(batch index, first key, first query) of each sequence; (batch, keys, queries) of the tensors; what the problem says of the lengths."""
    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    ends_k, ends_q, wide_k, wide_q = [0], [0], [0], [0]
    for nk, nq in LENGTHS:
        ends_k.append(ends_k[-1] + nk)
        ends_q.append(ends_q[-1] + nq)
        wide_k.append(wide_k[-1] + nk + 24)
        wide_q.append(wide_q[-1] + nq + 9)
    kw = dict(cu_seqlens_q=ints(ends_q), cu_seqlens_k=ints(ends_k), max_seqlen_q=MAX_Q, max_seqlen_k=MAX_K)
    if layout == "padded":
        return [(z, 0, 0) for z in range(len(LENGTHS))], (len(LENGTHS), MAX_K + 21, MAX_Q), dict(kw, varlen_type=cabi.VARLEN_PADDED)
    if layout == "strided":
        return [(0, k, q) for k, q in zip(wide_k, wide_q)], (1, wide_k[-1] + 5, wide_q[-1]), dict(kw, seq_strides_q=ints(wide_q), seq_strides_k=ints(wide_k))
    return [(0, k, q) for k, q in zip(ends_k, ends_q)], (1, ends_k[-1] + 37, ends_q[-1]), kw


def _want(q, k, v, do, scale, columns, rounded_shares):
    """Gradient of the shared columns of one sequence in 64 bits, (keys, columns), and how far it may be off.  Half a step (u) each: the forward's weights and its output,
    whose product with dO enters dS; dS; the result; and (rounded_shares) each kv head's share.  fp16 below its normal range: half its smallest step.  In 32 bits: scores
    of d products, twice in a weight; sums of dv, of the queries' and of the heads' terms; 8 more roundings, exponentials among them."""
    u, least = (2.0 ** -22, 0.0) if k.dtype == torch.float32 else (torch.finfo(k.dtype).eps / 2, 2.0 ** -25 if k.dtype == torch.float16 else 0.0)
    h, hk, d = q.shape[0], k.shape[0], q.shape[2]
    q, k, v, do = (t.double() for t in (q, k, v, do))
    k, v = k.repeat_interleave(h // hk, 0), v.repeat_interleave(h // hk, 0)
    x = q @ k.transpose(1, 2) * scale
    hidden = torch.ones(x.shape[-2:], dtype=torch.bool, device=x.device).triu(1)
    p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
    o, dp = p @ v, do @ v.transpose(1, 2)
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    mixed = p @ v.abs()
    terms = p * (do.abs() @ v.abs().transpose(1, 2) + (do.abs() * mixed).sum(-1, keepdim=True))      # what dS is the difference of
    output = u * (mixed + o.abs()) + least * (v.abs().sum(1, keepdim=True) + 1)
    score = ((d + 8) * 2.0 ** -24 * scale * (q.abs() @ k.abs().transpose(1, 2)) + (x.abs() + 8) * 2.0 ** -23).masked_fill(hidden, 0).amax(-1, keepdim=True)
    off = 1.05 * u * ds.abs() + 1.05 * p * (do.abs() * output).sum(-1, keepdim=True) + (3 * score + (v.shape[2] + 8) * 2.0 ** -23) * terms + least
    share = (ds.transpose(1, 2) @ q)[..., -columns:] * scale
    w = share.sum(0)
    most = (off.transpose(1, 2) @ q.abs())[..., -columns:].sum(0) * scale + (x.shape[1] + h) * 2.0 ** -24 * (ds.abs().transpose(1, 2) @ q.abs())[..., -columns:].sum(0) * scale
    if rounded_shares:
        most = most + 1.05 * u * share.unflatten(0, (hk, -1)).sum(1).abs().sum(0) + hk * least
    return w, most + 1.05 * u * (w.abs() + most) + least


@pytest.mark.parametrize("layout", ["compact", "strided", "padded"])
@pytest.mark.parametrize("dn,dr,dv,tail", DIMS)
@pytest.mark.parametrize("dtype", HALF + [torch.float32])
def test_rows_of_no_sequence_are_zero(dtype, dn, dr, dv, tail, layout):
    h, hk, d, scale = 4, 2, dn + dr, (dn + dr) ** -0.5
    places, (b, nk, nq), kw = _places(layout)
    g = torch.Generator(device="cuda").manual_seed(2)

    def rand(heads, tokens, width):
        return torch.randn(b, heads, tokens, width, generator=g, device="cuda").to(dtype)

    def holding_nan(t):
        return torch.full_like(t, math.nan)

    q, k, v, do = rand(h, nq, d), rand(hk, nk, d), rand(hk, nk, dv), rand(h, nq, dv)
    k[..., dn:] = k[:, :1, :, dn:]
    kw.update(sm_scale=scale, causal_type=1)
    out, lse = torch.zeros_like(do), torch.zeros(b * h, nq, device="cuda")
    assert cabi.attn_fwd(q, k, v, out, lse, **kw) == 0
    dq, dk, dv_ = holding_nan(q), holding_nan(k), holding_nan(v)
    args = (q, k, v, out, do, dq, dk, dv_, lse, torch.empty_like(lse))
    need = cabi.attn_bwd_shared_workspace(*args, dr, **kw)
    assert need == (b * hk * nk * dr if tail and dtype != torch.float32 else 0)
    workspace = torch.full([max(need, 4)], math.nan, device="cuda")
    shared = torch.full((b, 1, nk, dr), math.nan, device="cuda", dtype=dtype)
    assert cabi.attn_bwd_shared(*args, shared, workspace=workspace, **kw) == 0
    inside = torch.zeros(b, nk, dtype=torch.bool, device="cuda")
    for (z, k0, q0), (mk, mq) in zip(places, LENGTHS):
        inside[z, k0:k0 + mk] = True
        if not mk:
            continue
        got = shared[z, 0, k0:k0 + mk].double()
        if not mq:
            assert (got == 0).all()
            continue
        w, most = _want(q[z, :, q0:q0 + mq], k[z, :, k0:k0 + mk], v[z, :, k0:k0 + mk], do[z, :, q0:q0 + mq], scale, dr, not tail)
        assert ((got - w).abs() <= most + 1e-30).all(), float((got - w).abs().max())
    assert (shared[:, 0][~inside] == 0).all()


@pytest.mark.parametrize("layout", ["dense", "compact", "padded"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_problem_without_queries(dtype, layout):
    """No kernel runs, dK is left as it is, and nothing of it is summed."""
    h, hk, d, dv, dr, nk = 4, 2, 192, 128, 64, 40
    q, k, v, do = (torch.randn(1, n, s, w, device="cuda").to(dtype) for n, s, w in ((h, 5, d), (hk, nk, d), (hk, nk, dv), (h, 5, dv)))
    dq, dk, dv_ = (torch.full_like(t, math.nan) for t in (q, k, v))
    lse, delta = (torch.zeros(h, 5, device="cuda") for _ in range(2))
    kw = dict(sm_scale=0.1)
    if layout != "dense":
        ends = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 0], [0, nk])]
        kw.update(cu_seqlens_q=ends[0], cu_seqlens_k=ends[1], max_seqlen_q=0, max_seqlen_k=nk, varlen_type=cabi.VARLEN_PADDED if layout == "padded" else cabi.VARLEN_COMPACT)
    a = cabi.make_bwd_args(q, k, v, do, do, dq, dk, dv_, lse, delta, **kw)
    a.prob.max_seqlen_q = 0
    shared = torch.full((1, 1, nk, dr), math.nan, device="cuda", dtype=dtype)
    L, stream = cabi.lib(), cabi.current_stream_handle()
    need = L.ab200_attn_bwd_shared_workspace(a, dr, stream)
    assert need >= 0
    workspace = torch.full([max(need, 4)], math.nan, device="cuda")
    assert L.ab200_attn_bwd_shared(a, dr, cabi.view4(shared), workspace.data_ptr(), need, stream) == 0
    assert (shared == 0).all()
