"""The learned relative position bias and its table's gradient, against the 64-bit oracle.

The forward moves table entries and rounds each once, so it is compared bit for bit.  The gradient's sums are compared exactly where every
partial sum is a whole number below 2^24 (small whole gradients), and elsewhere within the rounding of a fp32 sum: every entry passes
through at most `adds` additions, each off by 2^-24 of a partial sum no larger than the sum of magnitudes, and the result is rounded
once to the table's type.  adds: at most 512 rows of each batch element in a thread, 40 in a CTA's sums, 1 for each 128 CTAs and 10 among
them.
"""
import pytest
import torch

from oracle import layer as O

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _tolerance(grad, where, buckets, dtype, want):
    adds = 512 * grad.shape[0] + 60 + grad.shape[0] * (grad.shape[2] + grad.shape[3]) // 128
    return adds * 2.0 ** -24 * O.relative_bias_grad(grad.abs(), where, buckets) + torch.finfo(dtype).eps / 2 * want.abs() * 1.001 + 1e-30


@pytest.mark.parametrize("dt,table_dt", [(BF16, BF16), (F16, F32), (F32, F32), (F32, BF16), (BF16, F16)])
@pytest.mark.parametrize("B,H,Sq,Sk,buckets,far,both,offset", [
    (1, 1, 1, 1, 32, 128, True, 0),
    (1, 3, 1, 777, 32, 128, False, 776),
    (2, 2, 7, 1, 16, 500, True, 3),
    (3, 2, 63, 65, 32, 128, True, -9),
    (2, 1, 64, 512, 64, 64, False, 0),      # buckets without a distance
    (2, 3, 65, 513, 4, 2, True, 100),
    (1, 2, 200, 1031, 32, 128, False, 5),
    (5, 1, 700, 90, 2, 3, False, -650),
    (1, 1, 8, 2048, 256, 2000, True, 1000),
])
def test_against_the_oracle(B, H, Sq, Sk, buckets, far, both, offset, dt, table_dt):
    from aotriton_b200 import autograd
    g = torch.Generator().manual_seed(Sq * 7 + Sk)
    table = torch.randn(buckets, H, generator=g).to(table_dt)
    where = O.bucket_matrix(Sq, Sk, buckets, far, both, offset)
    t = table.cuda().requires_grad_()
    bias = autograd.relative_position_bias(t, Sq, Sk, batch=B, max_distance=far, bidirectional=both, query_offset=offset, dtype=dt)
    assert bias.shape == (B, H, Sq, Sk) and bias.dtype == dt and bias.stride(0) == 0 and (bias.stride(2) * bias.element_size()) % 32 == 0
    want = O.relative_bias(table, where).to(dt)
    assert torch.equal(bias.detach().cpu(), want.expand(B, -1, -1, -1))
    # whole numbers: every sum is exact
    grad = torch.randint(-3, 4, (B, H, Sq, Sk), generator=g)
    got, = torch.autograd.grad(bias, t, grad.to(dt).cuda(), retain_graph=True)
    assert torch.equal(got.cpu(), O.relative_bias_grad(grad, where, buckets).to(table_dt))
    grad = torch.randn(B, H, Sq, Sk, generator=g).to(dt)
    got, = torch.autograd.grad(bias, t, grad.cuda())
    want = O.relative_bias_grad(grad, where, buckets)
    assert bool(((got.cpu().double() - want).abs() <= _tolerance(grad, where, buckets, table_dt, want)).all())


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("how", ["odd", "transposed", "sliced", "broadcast", "shifted"])
def test_gradients_of_any_layout(how, dt):
    from aotriton_b200 import autograd
    B, H, Sq, Sk = 2, 3, 130, 263
    g = torch.Generator().manual_seed(5)
    where = O.bucket_matrix(Sq, Sk, 32, 128, True, 0)
    whole = torch.randint(-3, 4, (B, H, Sq, Sk), generator=g).to(dt)
    if how == "odd":
        grad = whole.cuda()
    elif how == "transposed":
        grad = whole.cuda().transpose(2, 3).contiguous().transpose(2, 3)
    elif how == "sliced":
        grad = torch.full((B, H, Sq, 280), float("nan"), dtype=dt, device="cuda")[..., 8:8 + Sk]
        grad.copy_(whole)
    elif how == "shifted":
        grad = torch.full((B, H, Sq, 280), float("nan"), dtype=dt, device="cuda")[..., 3:3 + Sk]
        grad.copy_(whole)
    else:
        whole = whole[:1, :, :1].expand(B, H, Sq, Sk)
        grad = whole[:1, :, :1].cuda().expand(B, H, Sq, Sk)
    t = torch.randn(32, H, device="cuda").requires_grad_()
    got, = torch.autograd.grad(autograd.relative_position_bias(t, Sq, Sk, batch=B, dtype=dt), t, grad)
    assert torch.equal(got.cpu().double(), O.relative_bias_grad(whole, where, 32))


def test_views_beyond_the_entry_point():
    """The C entry: strides of every kind, and nothing written beside the bias."""
    from aotriton_b200 import autograd, cabi
    H, Sq, Sk = 2, 70, 531
    borders = autograd.relative_position_borders(16, 128)
    table = torch.randn(H, 40, device="cuda")[:, :32].t()      # (buckets, heads), neither stride 1
    want = O.relative_bias(table.cpu(), O.bucket_matrix(Sq, Sk, 32, 128, True, 0)).float()
    store = torch.full((H, Sq + 3, Sk + 8), 7.0, device="cuda")
    inner = torch.full((H, Sq, Sk, 2), 7.0, device="cuda")
    for view, rest in ((store[None, :, 1:1 + Sq, 4:4 + Sk], store), (store[None, :, 1:1 + Sq, 3:3 + Sk], store), (inner[None, ..., 0], inner)):
        rest.fill_(7.0)
        assert cabi.relative_bias_fwd(table, view, borders) == 0
        assert torch.equal(view[0].cpu(), want)
        view.fill_(7.0)
        assert bool((rest == 7.0).all())


def test_not_finite():
    """A NaN or infinity in the gradient reaches its own bucket's sum and no other."""
    from aotriton_b200 import autograd
    where = O.bucket_matrix(40, 300, 32, 128, True, 0)
    for dt in (F16, F32):
        for sk in (300, 296):
            t = torch.randn(32, 2, device="cuda").requires_grad_()
            grad = torch.ones(1, 2, 40, sk, device="cuda", dtype=dt)
            grad[0, 1, 11, 290], grad[0, 0, 3, 2] = float("nan"), float("inf")
            got, = torch.autograd.grad(autograd.relative_position_bias(t, 40, sk, dtype=dt), t, grad)
            bad = ~torch.isfinite(got.cpu())
            expected = torch.zeros(32, 2, dtype=torch.bool)
            expected[where[11, 290], 1] = expected[where[3, 2], 0] = True
            assert torch.equal(bad, expected)


def test_derivative_of_the_gradient_and_graph():
    from aotriton_b200 import autograd
    t = torch.randn(32, 2, device="cuda").requires_grad_()
    grad = torch.randn(1, 2, 33, 50, device="cuda").requires_grad_()
    first, = torch.autograd.grad(autograd.relative_position_bias(t, 33, 50), t, grad, create_graph=True)
    back = torch.randn(32, 2, device="cuda")
    second, = torch.autograd.grad(first, grad, back)      # the gradient is linear in `grad`: its derivative is the bias of `back`
    assert torch.equal(second[0].cpu().double(), O.relative_bias(back.cpu(), O.bucket_matrix(33, 50, 32, 128, True, 0)))

    def step():
        bias = autograd.relative_position_bias(t, 33, 50, batch=2)
        return bias.detach(), torch.autograd.grad(bias, t, torch.ones(2, 2, 33, 50, device="cuda"))[0]

    want = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        t.add_(1.0)
    graph.replay()
    assert torch.equal(got[0], want[0] + 1.0) or torch.allclose(got[0], want[0] + 1.0)
    assert torch.equal(got[1], want[1])


def test_same_bits_every_time_and_on_other_streams():
    from aotriton_b200 import autograd
    t = torch.randn(32, 4, device="cuda").requires_grad_()
    grad = torch.randn(3, 4, 500, 517, device="cuda", dtype=BF16)
    bias = autograd.relative_position_bias(t, 500, 517, batch=3, dtype=BF16)
    first, = torch.autograd.grad(bias, t, grad, retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both = [torch.autograd.grad(autograd.relative_position_bias(t, 500, 517, batch=3, dtype=BF16), t, grad)[0] for _ in range(3)]
    again = [torch.autograd.grad(bias, t, grad, retain_graph=True)[0] for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in both + again)


def test_python_way_equals_the_native_one():
    from aotriton_b200 import autograd
    t = torch.randn(32, 4, device="cuda").requires_grad_()
    grad = torch.randn(3, 4, 50, 67, device="cuda", dtype=F16)
    native = autograd.relative_position_bias(t, 50, 67, batch=3, dtype=F16)
    python = autograd._RelativeBias.apply(t, 50, 67, 3, autograd.relative_position_borders(16, 128), True, 0, F16)
    assert torch.equal(native, python) and native.stride() == python.stride()
    assert torch.equal(torch.autograd.grad(native, t, grad)[0], torch.autograd.grad(python, t, grad)[0])


def test_empty():
    from aotriton_b200 import autograd
    t = torch.randn(32, 4, device="cuda").requires_grad_()
    for sq, sk, b in ((0, 5, 1), (5, 0, 1), (5, 5, 0)):
        bias = autograd.relative_position_bias(t, sq, sk, batch=b)
        assert bias.shape == (b, 4, sq, sk)
        got, = torch.autograd.grad(bias, t, torch.ones_like(bias))
        assert bool((got == 0).all())


def test_offsets_beyond_32_bits():
    """More than 2^31 entries: what the last rows hold, and a gradient that only they have."""
    from aotriton_b200 import autograd
    S, buckets, far, rows = 50001, 32, 128, 3
    table = torch.randn(buckets, 1, device="cuda").to(BF16).requires_grad_()
    bias = autograd.relative_position_bias(table, S, S, max_distance=far)
    where = O.bucket_matrix(rows, S, buckets, far, True, S - rows)
    assert torch.equal(bias[0, 0, -rows:].detach().cpu(), table.detach().cpu()[where][..., 0])
    grad = torch.zeros(1, 1, S, S, device="cuda", dtype=BF16)
    last = torch.randint(-1, 2, (rows, S), generator=torch.Generator().manual_seed(3))
    grad[0, 0, -rows:] = last.to(BF16).cuda()
    got, = torch.autograd.grad(bias, table, grad)
    want = O.relative_bias_grad(last[None, None], where, buckets)      # (whole numbers, rounded once)
    assert torch.equal(got.cpu(), want.to(BF16))
