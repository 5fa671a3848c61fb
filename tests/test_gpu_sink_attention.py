"""Attention with a sliding window and first keys that stay visible, forward and backward, against the 64-bit reference and its bound
(_sink_reference.py): block, tile and window boundaries, few queries against long caches, queries ahead of all keys, packed and padded
batches, every kernel family."""
import pytest
import torch

from _sink_reference import check, reference

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rand(*shapes, dt, seed=0, layout="bhsd"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda b, h, s, d: (torch.randn(b, s, h, d, generator=g, device="cuda").to(dt).transpose(1, 2) if layout == "bshd"
                               else torch.randn(b, h, s, d, generator=g, device="cuda").to(dt))
    return [make(*s) for s in shapes]


def _healthy():
    from aotriton_b200 import cabi
    torch.cuda.synchronize()
    assert cabi.lib().ab200_kernel_status(0) == 0


def _family(dt, d, dv):
    return 2 if dt != F32 and max(d, dv) <= 256 and d % 8 == 0 and dv % 8 == 0 else 1


FORWARD_BACKWARD = [
    # B, Hq, Hk, Sq, Sk, D, Dv, window, sinks
    (1, 1, 1, 1, 1, 64, 64, 1, 0),
    (1, 2, 2, 17, 17, 64, 64, 3, 1),
    (1, 2, 1, 256, 256, 128, 128, 64, 4),        # whole tiles
    (1, 2, 1, 256, 256, 64, 64, 1, 128),         # the first block all first keys, a window of one
    (2, 4, 2, 300, 300, 64, 64, 37, 5),
    (1, 2, 1, 700, 700, 128, 128, 129, 200),     # first keys that end inside their second block
    (1, 2, 2, 513, 513, 128, 64, 128, 127),
    (1, 4, 2, 384, 384, 128, 128, 200, 0),       # a window alone
    (1, 2, 1, 200, 200, 128, 128, 500, 3),       # nothing out of sight
    (1, 2, 1, 200, 200, 64, 64, 150, 60),
    (1, 2, 1, 100, 900, 128, 128, 64, 4),        # the last queries of longer keys
    (1, 2, 2, 130, 1000, 64, 64, 300, 700),
    (1, 2, 1, 200, 90, 128, 128, 16, 4),         # queries ahead of all keys see nothing
    (1, 8, 1, 1500, 1500, 128, 128, 64, 4),      # the first keys' queries shared out, one kv head for eight
    (2, 2, 2, 1537, 1537, 64, 64, 100, 33),
    (1, 3, 3, 260, 260, 72, 72, 50, 4),          # padded and unequal head dims
    (1, 2, 1, 260, 260, 40, 96, 50, 4),
    (1, 2, 1, 300, 300, 256, 256, 70, 5),        # wide heads
    (1, 2, 2, 512, 512, 256, 256, 64, 64),
    (1, 4, 2, 200, 700, 160, 200, 100, 66),
]


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("case", FORWARD_BACKWARD, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_gradients(case, dt):
    from aotriton_b200 import autograd, cabi
    B, Hq, Hk, Sq, Sk, D, Dv, window, sinks = case
    q, k, v, do = _rand((B, Hq, Sq, D), (B, Hk, Sk, D), (B, Hk, Sk, Dv), (B, Hq, Sq, Dv), dt=dt, seed=Sq + Sk + D, layout="bshd" if Sq % 2 else "bhsd")
    for t in (q, k, v):
        t.requires_grad_()
    out, lse = autograd.sink_attention(q, k, v, window, sinks, return_lse=True)
    grads = torch.autograd.grad(out, (q, k, v), do)
    assert autograd.last_bwd_family == _family(dt, D, Dv)
    values, bounds = reference(q.detach(), k.detach(), v.detach(), window, sinks, D ** -0.5, do)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out.detach(), lse) + grads):
        check(name, got, values, bounds)
    # without a gradient, and without the log-sum-exp
    with torch.no_grad():
        again = autograd.sink_attention(q, k, v, window, sinks)
        assert torch.equal(again, out) and cabi.lib().ab200_last_fwd_family() == _family(dt, D, Dv)
    _healthy()


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128, 300, 52])
@pytest.mark.parametrize("Hq,Hk,Sq", [(8, 2, 1), (4, 4, 3), (16, 1, 16), (3, 3, 2)])
@pytest.mark.parametrize("Sk,window,sinks", [(1, 1, 0), (5, 2, 1), (63, 7, 4), (64, 16, 1), (65, 1, 65), (129, 64, 64), (500, 100, 70), (2100, 64, 3), (6007, 2000, 4),
                                             (2500, 1, 2000)])
def test_few_queries_against_a_cache(Hq, Hk, Sq, Sk, window, sinks, D, dt):
    from aotriton_b200 import autograd
    q, k, v = _rand((2, Hq, Sq, D), (2, Hk, Sk, D), (2, Hk, Sk, D), dt=dt, seed=Sk + Sq)
    out, lse = autograd.sink_attention(q, k, v, window, sinks, return_lse=True)
    values, bounds = reference(q, k, v, window, sinks, D ** -0.5)
    check("out", out, values, bounds)
    check("lse", lse, values, bounds)
    _healthy()


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Sq", [1, 5, 40, 130])
def test_what_nobody_sees_may_hold_anything(Sq, D, dt):
    """Keys between the first ones and the first query's window: NaN and infinities there change no bit of out, lse and dq."""
    from aotriton_b200 import autograd
    Sk, window, sinks = 1500, 200, 5
    q, k, v, do = _rand((1, 4, Sq, D), (1, 2, Sk, D), (1, 2, Sk, D), (1, 4, Sq, D), dt=dt, seed=Sq)
    q.requires_grad_()
    dirty_k, dirty_v = k.clone(), v.clone()
    hidden = slice(sinks, Sk - Sq - window + 1)
    dirty_k[:, :, hidden] = float("nan")
    dirty_v[:, :, hidden] = float("inf")
    dirty_v[:, :, hidden.stop - 3] = float("nan")
    results = []
    for kk, vv in ((k, v), (dirty_k, dirty_v)):
        out, lse = autograd.sink_attention(q, kk, vv, window, sinks, return_lse=True)
        results.append([out.detach(), lse, torch.autograd.grad(out, q, do)[0]])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    values, bounds = reference(q.detach(), k, v, window, sinks, D ** -0.5, do)
    check("dq", results[1][2], values, bounds)
    _healthy()


def _ends(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F16, 256), (F32, 64), (BF16, 60)])
@pytest.mark.parametrize("lens_q,lens_k", [([5, 0, 300, 129, 1], None), ([1, 16, 3], [700, 16, 90]), ([200, 7, 128], [450, 5, 0]), ([600, 900], None)])
def test_packed(lens_q, lens_k, dt, D):
    from aotriton_b200 import autograd
    lens_k = lens_k or lens_q
    Hq, Hk, window, sinks = 4, 2, 60, 6
    tq, tk = sum(lens_q), sum(lens_k)
    q, k, v, do = _rand((1, Hq, tq, D), (1, Hk, tk, D), (1, Hk, tk, D), (1, Hq, tq, D), dt=dt, seed=tq, layout="bshd")
    for t in (q, k, v):
        t.requires_grad_()
    out, lse = autograd.varlen_sink_attention(q, k, v, _ends(lens_q), _ends(lens_k), max(lens_q), max(lens_k), window, sinks, return_lse=True)
    grads = torch.autograd.grad(out, (q, k, v), do)
    at_q = at_k = 0
    for nq, nk in zip(lens_q, lens_k):
        sl_q, sl_k = slice(at_q, at_q + nq), slice(at_k, at_k + nk)
        at_q, at_k = at_q + nq, at_k + nk
        if not nq:
            assert bool((grads[1][:, :, sl_k] == 0).all()) and bool((grads[2][:, :, sl_k] == 0).all())
            continue
        if not nk:
            assert bool((out[:, :, sl_q] == 0).all()) and bool(torch.isinf(lse[:, sl_q]).all()) and bool((grads[0][:, :, sl_q] == 0).all())
            continue
        part = [t.detach()[:, :, sl] for t, sl in ((q, sl_q), (k, sl_k), (v, sl_k))]
        values, bounds = reference(*part, window, sinks, D ** -0.5, do[:, :, sl_q])
        for name, got in (("out", out.detach()[:, :, sl_q]), ("lse", lse[:, sl_q]), ("dq", grads[0][:, :, sl_q]), ("dk", grads[1][:, :, sl_k]),
                          ("dv", grads[2][:, :, sl_k])):
            check(name, got, values, bounds)
    _healthy()


@pytest.mark.parametrize("dt,D", [(BF16, 128), (F16, 64), (F16, 256), (F32, 64), (F32, 160), (BF16, 60)])
@pytest.mark.parametrize("Sq,Sk,lens_q,lens_k", [(1, 900, [1, 1, 0, 1], [900, 65, 300, 1]), (8, 400, [8, 3, 0, 5], [400, 3, 77, 260]),
                                                 (300, 300, [300, 0, 1, 257], [300, 0, 1, 257]), (100, 500, [100, 40, 100, 7], [500, 90, 0, 130])])
def test_padded(Sq, Sk, lens_q, lens_k, dt, D):
    """A batch of caches: what lies behind the sequences is NaN, and comes out as zero."""
    from aotriton_b200 import autograd
    B, Hq, Hk, window, sinks = len(lens_q), 4, 2, 50, 5
    q, k, v, do = _rand((B, Hq, Sq, D), (B, Hk, Sk, D), (B, Hk, Sk, D), (B, Hq, Sq, D), dt=dt, seed=Sk)
    for z, (nq, nk) in enumerate(zip(lens_q, lens_k)):
        q[z, :, nq:] = float("nan")
        k[z, :, nk:] = v[z, :, nk:] = float("nan")
        do[z, :, nq:] = float("nan")
    for t in (q, k, v):
        t.requires_grad_()
    out, lse = autograd.varlen_sink_attention(q, k, v, _ends(lens_q), _ends(lens_k), max(lens_q), max(lens_k), window, sinks, return_lse=True, varlen_type="padded")
    assert lse.shape == (B * Hq, Sq)
    grads = torch.autograd.grad(out, (q, k, v), do)
    lse = lse.view(B, Hq, Sq)
    for z, (nq, nk) in enumerate(zip(lens_q, lens_k)):
        assert bool((out[z, :, nq:] == 0).all()) and bool((lse[z, :, nq:] == float("inf")).all())
        assert all(bool((t[z, :, n:] == 0).all()) for t, n in zip(grads, (nq, nk, nk)))
        if not nq or not nk:
            assert bool((out[z] == 0).all()) and all(bool((t[z] == 0).all()) for t in grads)
            continue
        part = [t.detach()[z:z + 1, :, :n] for t, n in ((q, nq), (k, nk), (v, nk))]
        values, bounds = reference(*part, window, sinks, D ** -0.5, do[z:z + 1, :, :nq])
        for name, got in (("out", out.detach()[z, :, :nq]), ("lse", lse[z, :, :nq]), ("dq", grads[0][z, :, :nq]), ("dk", grads[1][z, :, :nk]),
                          ("dv", grads[2][z, :, :nk])):
            check(name, got, values, bounds)
    _healthy()


@pytest.mark.parametrize("dt,D,S", [(BF16, 128, 640), (F16, 256, 300), (F32, 64, 200)])
def test_same_bits_on_other_streams_in_graphs_and_by_python(dt, D, S):
    from aotriton_b200 import autograd
    q, k, v, do = _rand((2, 4, S, D), (2, 2, S, D), (2, 2, S, D), (2, 4, S, D), dt=dt)
    for t in (q, k, v):
        t.requires_grad_()

    def step(f=lambda: autograd.sink_attention(q, k, v, 70, 5)):
        out = f()
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), do)

    want = step()
    runs = [step() for _ in range(3)]
    runs.append(step(lambda: autograd._SinkAttention.apply(q, k, v, None, None, 0, 0, 70, 5, D ** -0.5, False, 0)))
    side = [torch.cuda.Stream() for _ in range(2)]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):      # two streams at once
        for s in side:
            with torch.cuda.stream(s):
                runs.append(step())
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    torch.cuda.synchronize()
    for _ in range(2):      # two captured steps side by side
        for s, (graph, _) in zip(side, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for got in runs + [r for _, r in graphs]:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    _healthy()


def test_gradient_layouts_and_second_derivative():
    from aotriton_b200 import autograd
    q, k, v, do = _rand((1, 4, 200, 64), (1, 2, 200, 64), (1, 2, 200, 64), (1, 4, 200, 64), dt=F16)
    for t in (q, k, v):
        t.requires_grad_()
    out = autograd.sink_attention(q, k, v, 30, 3)
    want = torch.autograd.grad(out, (q, k, v), do, retain_graph=True)
    odd = do.transpose(2, 3).contiguous().transpose(2, 3)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, (q, k, v), odd, retain_graph=True), want))
    got = torch.autograd.grad(out.sum(), (q, k, v), retain_graph=True)
    ones = torch.autograd.grad(out, (q, k, v), torch.ones_like(out), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, ones))
    first = torch.autograd.grad(out, q, do, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(first.sum(), q)
    # q without a unit innermost stride
    odd = q.detach().transpose(2, 3).contiguous().transpose(2, 3).requires_grad_()
    out2 = autograd.sink_attention(odd, k, v, 30, 3)
    assert torch.equal(out2, out) and torch.equal(torch.autograd.grad(out2, odd, do)[0], want[0])


def test_empty():
    from aotriton_b200 import autograd
    for shape in ((0, 4, 2, 5, 5), (1, 4, 2, 0, 5), (1, 4, 2, 5, 0)):
        B, Hq, Hk, Sq, Sk = shape
        q, k, v = (torch.ones(B, h, s, 64, device="cuda", dtype=F16, requires_grad=True) for h, s in ((Hq, Sq), (Hk, Sk), (Hk, Sk)))
        out, lse = autograd.sink_attention(q, k, v, 3, 1, return_lse=True)
        assert out.shape == (B, Hq, Sq, 64) and bool((out == 0).all()) and bool(torch.isinf(lse).all())
        for g, t in zip(torch.autograd.grad(out, (q, k, v), torch.ones_like(out)), (q, k, v)):
            assert g.shape == t.shape and bool((g == 0).all())


def test_long_cache_offsets():
    """Tensors of more than 2^31 elements: one token near the end of a long cache, far behind the first keys."""
    from aotriton_b200 import autograd
    Hk, Sk, D, window, sinks = 8, 2_200_000, 128, 300, 4
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.zeros(1, Hk, Sk, D, device="cuda", dtype=BF16) for _ in range(2))
    for t in (k, v):
        t[:, :, :64] = torch.randn(1, Hk, 64, D, generator=g, device="cuda").to(BF16)
        t[:, :, -400:] = torch.randn(1, Hk, 400, D, generator=g, device="cuda").to(BF16)
    q = torch.randn(1, 16, 1, D, generator=g, device="cuda").to(BF16)
    out = autograd.sink_attention(q, k, v, window, sinks)
    near_k, near_v = (torch.cat([t[:, :, :sinks], t[:, :, -window:]], 2) for t in (k, v))
    values, bounds = reference(q, near_k, near_v, window + sinks, 0, D ** -0.5)
    check("out", out, values, bounds)
    _healthy()


@pytest.mark.parametrize("dt,D,layout", [(BF16, 128, "bshd"), (F16, 64, "bhsd"), (F16, 256, "bshd"), (F32, 64, "bshd"), (F32, 160, "bhsd"), (BF16, 60, "bshd")])
@pytest.mark.parametrize("lens_q,lens_k", [([200, 7, 128], None), ([1, 1, 1], [300, 90, 1]), ([0, 0], [0, 0])])
def test_packed_with_room_behind(lens_q, lens_k, dt, D, layout):
    """Tokens behind the last sequence, as where buffers have one size for all batches: NaN there reaches nothing, and comes out as zero."""
    from aotriton_b200 import autograd
    lens_k = lens_k or lens_q
    Hq, Hk, window, sinks, room = 4, 2, 60, 6, 75
    tq, tk = sum(lens_q), sum(lens_k)
    q, k, v, do = _rand((1, Hq, tq + room, D), (1, Hk, tk + room, D), (1, Hk, tk + room, D), (1, Hq, tq + room, D), dt=dt, seed=tq, layout=layout)
    for t, n in ((q, tq), (k, tk), (v, tk), (do, tq)):
        t[:, :, n:] = float("nan")
    for t in (q, k, v):
        t.requires_grad_()
    max_q, max_k = max(*lens_q, 1), max(*lens_k, 1)
    args = (_ends(lens_q), _ends(lens_k), max_q, max_k, window, sinks)
    junk = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(8)]      # (what fresh tensors may hold)
    del junk
    for native in (True, False):
        if native:
            out, lse = autograd.varlen_sink_attention(q, k, v, *args, return_lse=True)
        else:
            out, lse = autograd._SinkAttention.apply(q, k, v, *args, D ** -0.5, True, 1)
        grads = torch.autograd.grad(out, (q, k, v), do)
        assert lse.shape == (Hq, tq + room)
        assert bool((out[:, :, tq:] == 0).all()) and bool((lse[:, tq:] == float("inf")).all())
        assert all(bool((t[:, :, n:] == 0).all()) for t, n in zip(grads, (tq, tk, tk)))
        at_q = at_k = 0
        for nq, nk in zip(lens_q, lens_k):
            sl_q, sl_k = slice(at_q, at_q + nq), slice(at_k, at_k + nk)
            at_q, at_k = at_q + nq, at_k + nk
            if not nq:
                continue
            part = [t.detach()[:, :, sl] for t, sl in ((q, sl_q), (k, sl_k), (v, sl_k))]
            values, bounds = reference(*part, window, sinks, D ** -0.5, do[:, :, sl_q])
            for name, got in (("out", out.detach()[:, :, sl_q]), ("lse", lse[:, sl_q]), ("dq", grads[0][:, :, sl_q]), ("dk", grads[1][:, :, sl_k]),
                              ("dv", grads[2][:, :, sl_k])):
                check(name, got, values, bounds)
    _healthy()


@pytest.mark.parametrize("dt,D", [(F32, 64), (F32, 128), (F32, 40), (BF16, 60), (F16, 124), (BF16, 256), (F16, 160)])
@pytest.mark.parametrize("window,sinks", [(30, 4), (100, 45)])
@pytest.mark.parametrize("lens_q,lens_k", [([1000], None), ([1000, 0, 3, 200], None), ([40, 900], [1000, 950])])
def test_first_keys_shared_by_many_queries(lens_q, lens_k, window, sinks, dt, D):
    """Register-tiled backward and wide heads: several CTAs share the queries of the first keys.  Short and empty sequences beside long ones."""
    from aotriton_b200 import autograd, cabi
    lens_k = lens_k or lens_q
    Hq, Hk = 8, 2
    tq, tk = sum(lens_q), sum(lens_k)
    q, k, v, do = _rand((1, Hq, tq, D), (1, Hk, tk, D), (1, Hk, tk, D), (1, Hq, tq, D), dt=dt, seed=tq + sinks, layout="bshd")
    for t in (q, k, v):
        t.requires_grad_()
    args = (_ends(lens_q), _ends(lens_k), max(lens_q), max(lens_k))
    out, lse = autograd.varlen_sink_attention(q, k, v, *args, window, sinks, return_lse=True)
    need = cabi.sink_attn_bwd_workspace(q, k, v, out, do, q, k, v, lse, torch.empty_like(lse), window, sinks, sm_scale=1.0, cu_seqlens_q=args[0],
                                        cu_seqlens_k=args[1], max_seqlen_q=args[2], max_seqlen_k=args[3], varlen_type=1)
    assert need > 0
    poison = torch.full((need,), float("nan"), device="cuda")      # (the workspace that the backward gets next)
    del poison
    grads = torch.autograd.grad(out, (q, k, v), do, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(out, (q, k, v), do)))
    at_q = at_k = 0
    for nq, nk in zip(lens_q, lens_k):
        sl_q, sl_k = slice(at_q, at_q + nq), slice(at_k, at_k + nk)
        at_q, at_k = at_q + nq, at_k + nk
        if not nq:
            assert bool((grads[1][:, :, sl_k] == 0).all()) and bool((grads[2][:, :, sl_k] == 0).all())
            continue
        part = [t.detach()[:, :, sl] for t, sl in ((q, sl_q), (k, sl_k), (v, sl_k))]
        values, bounds = reference(*part, window, sinks, D ** -0.5, do[:, :, sl_q])
        for name, got in (("out", out.detach()[:, :, sl_q]), ("dq", grads[0][:, :, sl_q]), ("dk", grads[1][:, :, sl_k]), ("dv", grads[2][:, :, sl_k])):
            check(name, got, values, bounds)
    _healthy()
