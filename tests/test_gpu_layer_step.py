"""The operators around attention run together, as a layer runs them: an encoder's step (relative position bias, attention with dropout,
dropout with the residual's addition) with every gradient against 64 bits, a decoder's training step, and a decoder's prompt and single tokens over a
padded cache by a captured step.

Bounds as in _sink_reference.py, carried from one operator to the next to first order; 1.02 covers the products of two of them (a rounding is at
most 2^-8, and fewer than five meet in any term).
"""
import numpy as np
import pytest
import torch

from _sink_reference import check, reference
from oracle import layer as O
from oracle import philox

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
T = lambda t: t.transpose(-1, -2)


def _encoder_reference(q, k, v, table, x, dy, where, sm_scale, p_attn, keep, p_hidden, keep_hidden):
    """(values, bounds) of y, dq, dk, dv, dtable; all in 64 bits on the CPU."""
    dt = q.dtype
    half, tiny = torch.finfo(dt).eps / 2 * 1.001, 2.0 ** -25 if dt == F16 else 0.0
    B, H, S, D = q.shape
    g = H // k.shape[1]
    merge = lambda t: t.transpose(1, 2).reshape(B, S, H * D)
    split = lambda t: t.view(B, S, H, D).transpose(1, 2)
    fold = lambda t: t.view(B, H // g, g, *t.shape[2:]).sum(2)
    Q, K, V = q.double(), k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    bias = O.relative_bias(table, where).to(dt).double()      # (moved and rounded once, as the operator does)
    p = torch.softmax((Q @ T(K)) * sm_scale + bias, -1)
    size = float(((Q.abs() @ T(K.abs())) * sm_scale + bias.abs()).max())
    slop = 2 * (D + 5) * 2.0 ** -24 * size + 2.0 ** -20 + S * 2.0 ** -24
    up, up_hidden = 1 / (1 - p_attn), 1 / (1 - p_hidden)
    kept = keep.double() * up
    out = (p * kept) @ V
    e_out = (half + slop) * ((p * kept) @ V.abs()) + tiny * (kept @ V.abs()) + half * out.abs()
    kh = keep_hidden.double().view(B, S, H * D) * up_hidden
    y = x.double() + kh * merge(out)
    e_y = kh * merge(e_out) + 4 * 2.0 ** -24 * (x.double().abs() + kh * merge(out).abs()) + half * y.abs()
    do = split(kh * dy.double())
    e_do = (half + 3 * 2.0 ** -24) * do.abs() + tiny
    dp = kept * (do @ T(V))
    e_dp = kept * (e_do @ T(V.abs()))
    dp_size = kept * (do.abs() @ T(V.abs()))
    delta = (out * do).sum(-1, keepdim=True)
    e_delta = (e_out * do.abs() + out.abs() * e_do + D * 2.0 ** -24 * (out * do).abs()).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_ds = half * ds.abs() + slop * p * (dp_size + delta.abs()) + p * (e_dp + e_delta) + tiny
    e_p = ((half + slop) * p + tiny) * kept
    n = g * S * 2.0 ** -24
    values = dict(y=y, dq=ds @ K * sm_scale, dk=fold(T(ds) @ Q) * sm_scale, dv=fold(T(p * kept) @ do), dtable=O.relative_bias_grad(ds, where, table.shape[0]))
    bounds = dict(y=e_y, dq=(e_ds @ K.abs() + n * (ds.abs() @ K.abs())) * sm_scale, dk=fold(T(e_ds) @ Q.abs() + n * (T(ds.abs()) @ Q.abs())) * sm_scale,
                  dv=fold(T(e_p) @ do.abs() + T(p * kept) @ e_do + n * (T(p * kept) @ do.abs())),
                  dtable=O.relative_bias_grad(e_ds + (60 + 512 * B) * 2.0 ** -24 * ds.abs(), where, table.shape[0]))
    for name in ("dq", "dk", "dv"):
        bounds[name] = bounds[name] + half * values[name].abs() + (2.0 ** -25 if dt == F16 else 1e-37)
    bounds["dtable"] = bounds["dtable"] + torch.finfo(table.dtype).eps / 2 * values["dtable"].abs() + 1e-30
    return values, {n: 1.02 * b for n, b in bounds.items()}


@pytest.mark.parametrize("dt,B,H,Hk,S,D,both", [(F16, 2, 4, 2, 150, 64, True), (BF16, 1, 3, 3, 257, 128, False), (F32, 2, 2, 1, 70, 64, True)])
def test_encoder_step(dt, B, H, Hk, S, D, both):
    from aotriton_b200 import autograd
    g = torch.Generator().manual_seed(S)
    q, x, dy = (torch.randn(s, generator=g).to(dt) for s in ((B, H, S, D), (B, S, H * D), (B, S, H * D)))
    k, v = (torch.randn(B, Hk, S, D, generator=g).to(dt) for _ in range(2))
    table = torch.randn(16, H, generator=g)
    p_attn, p_hidden, seed = 0.2, 0.1, 0x51EED
    leaves, on_device = [t.cuda().requires_grad_() for t in (q, k, v, table, x)], dy.cuda()

    def step(seed_hidden, offset_hidden):
        q_, k_, v_, t_, x_ = leaves
        bias = autograd.relative_position_bias(t_, S, S, batch=B, max_distance=64, bidirectional=both, dtype=dt)
        out = autograd.attention(q_, k_, v_, b=bias, dropout_p=p_attn, philox_seed=seed, philox_offset1=0)
        y = autograd.dropout(out.transpose(1, 2).reshape(B, S, H * D), p_hidden, residual=x_, philox_seed=seed_hidden, philox_offset=offset_hidden)
        return (y.detach(),) + torch.autograd.grad(y, leaves, on_device)

    got = step(seed, 1 << 40)
    base = autograd.DEFAULT_PHILOX_OFFSET_2
    keep = torch.from_numpy(np.stack([[philox.keep_mask(seed, base, z, h, H, S, S, S, S, p_attn) for h in range(H)] for z in range(B)]))
    where = O.bucket_matrix(S, S, 16, 64, both, 0)
    values, bounds = _encoder_reference(q, k, v, table, x, dy, where, D ** -0.5, p_attn, keep, p_hidden, O.dropout_keep(x.numel(), p_hidden, seed, 1 << 40))
    for name, t in zip(("y", "dq", "dk", "dv", "dtable"), got):
        check(name, t.cpu(), values, bounds)
    assert torch.equal(got[5], on_device)
    # the same step captured, its seeds in tensors
    numbers = [torch.tensor([n], dtype=torch.int64, device="cuda") for n in (seed, 1 << 40)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*numbers)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = step(*numbers)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, got))
    numbers[1].fill_(5)      # other keep bits at the next replay
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, step(seed, 5))) and not torch.equal(again[0], got[0])


@pytest.mark.parametrize("dt,Hq,Hk,S,D", [(BF16, 8, 2, 333, 128), (F16, 4, 4, 260, 64)])
def test_decoder_step(dt, Hq, Hk, S, D):
    """Sink attention, then dropout with the residual: the gradient that reaches attention is the dropout's output, bit for bit."""
    from aotriton_b200 import autograd
    g = torch.Generator().manual_seed(S)
    q, k, v, x, dy = (torch.randn(s, generator=g).to(dt).cuda() for s in ((1, Hq, S, D), (1, Hk, S, D), (1, Hk, S, D), (1, S, Hq * D), (1, S, Hq * D)))
    leaves = [t.requires_grad_() for t in (q, k, v, x)]
    out = autograd.sink_attention(q, k, v, 100, 4)
    y = autograd.dropout(out.transpose(1, 2).reshape(1, S, Hq * D), 0.1, residual=x, philox_offset=9)
    dq, dk, dv, dx = torch.autograd.grad(y, leaves, dy)
    do = autograd.dropout(dy, 0.1, philox_offset=9).view(1, S, Hq, D).transpose(1, 2)
    values, bounds = reference(q.detach(), k.detach(), v.detach(), 100, 4, D ** -0.5, do)
    for name, t in (("out", out.detach()), ("dq", dq), ("dk", dk), ("dv", dv)):
        check(name, t, values, bounds)
    assert torch.equal(dx, dy)


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64)])
def test_prompt_and_tokens_over_a_cache(dt, D):
    """Prompts of different lengths into a padded cache that holds NaN elsewhere, then tokens by one captured step: every row is the whole sequence's."""
    from aotriton_b200 import autograd
    Hq, Hk, room, window, sinks, steps = 8, 2, 700, 90, 3, 12
    prompts = [1, 97, 400, 640]
    B = len(prompts)
    q, k, v = (torch.randn(B, h, room, D, device="cuda").to(dt) for h in (Hq, Hk, Hk))
    ck, cv = (torch.full((B, Hk, room, D), float("nan"), device="cuda", dtype=dt) for _ in range(2))
    for z, n in enumerate(prompts):
        ck[z, :, :n], cv[z, :, :n] = k[z, :, :n], v[z, :, :n]
    lens = torch.tensor(prompts, device="cuda")
    ends = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    ends[1:] = lens.cumsum(0)
    out = autograd.varlen_sink_attention(q[:, :, :max(prompts)], ck, cv, ends, ends, max(prompts), room, window, sinks, varlen_type="padded")
    ones, rows = torch.arange(B + 1, dtype=torch.int32, device="cuda"), torch.arange(B, device="cuda")
    token, tk, tv = torch.empty(B, Hq, 1, D, device="cuda", dtype=dt), *(torch.empty(B, Hk, D, device="cuda", dtype=dt) for _ in range(2))

    def step():
        ck[rows, :, lens], cv[rows, :, lens] = tk, tv
        lens.add_(1)
        ends[1:] = lens.cumsum(0)
        return autograd.varlen_sink_attention(token, ck, cv, ones, ends, 1, room, window, sinks, varlen_type="padded")

    at = list(prompts)

    def fill():
        for z, n in enumerate(at):
            token[z, :, 0], tk[z], tv[z] = q[z, :, n], k[z, :, n], v[z, :, n]
            at[z] += 1

    results = [[out[z, :, :n]] for z, n in enumerate(prompts)]
    side = torch.cuda.Stream()
    fill()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        later = step()
    for z in range(B):
        results[z].append(first[z])
    for _ in range(steps - 1):
        fill()
        graph.replay()
        for z in range(B):
            results[z].append(later[z].clone())
    for z, n in enumerate(at):
        values, bounds = reference(q[z:z + 1, :, :n], k[z:z + 1, :, :n], v[z:z + 1, :, :n], window, sinks, D ** -0.5)
        check("out", torch.cat(results[z], 1), values, bounds)
    for z, n in enumerate(prompts):
        assert bool((out[z, :, n:] == 0).all())
