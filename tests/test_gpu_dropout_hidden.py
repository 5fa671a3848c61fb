"""Dropout of hidden states with the residual's addition, against the 64-bit oracle with the oracle's keep mask.

The tolerance counts the roundings: 1 / (1 - p) in fp32, its product with x and the sum, 2^-24 of their size each (3 * 2^-24 of
|x| / (1 - p) + |residual|), and one rounding to the tensor's type.
"""
import pytest
import torch

from oracle import layer as O

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _check(got, x, residual, keep, p):
    kept = x.double().cpu() / (1 - p) if p < 1 else torch.zeros_like(x.double().cpu())
    kept = torch.where(keep.view(x.shape), kept, 0.0)
    r = torch.zeros_like(kept) if residual is None else residual.double().cpu()
    want = kept + r
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps      # (half an ulp of a subnormal result)
    bound = torch.finfo(got.dtype).eps / 2 * want.abs() * 1.001 + 3 * 2.0 ** -24 * (kept.abs() + r.abs()) + tiny
    assert bool(((got.double().cpu() - want).abs() <= bound).all())
    if residual is None:
        assert bool((got.cpu()[~keep.view(x.shape)] == 0).all())


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1,), (3,), (5, 7), (2, 3, 64), (9, 1003), (4, 4096), (17, 8), (3, 2048), (1, 100001)])
@pytest.mark.parametrize("p,add", [(0.1, True), (0.5, False), (0.0, True), (0.0, False), (1.0, True), (1.0, False)])
def test_against_the_oracle(shape, p, add, dt):
    from aotriton_b200 import autograd
    g = torch.Generator().manual_seed(len(shape) + shape[-1])
    x, res, dy = (torch.randn(shape, generator=g).to(dt).cuda() for _ in range(3))
    x.requires_grad_()
    res = res.requires_grad_() if add else None
    seed, offset = 0x123456789ABC, 2 ** 32 - 3      # (the counter's low word runs over)
    y = autograd.dropout(x, p, residual=res, philox_seed=seed, philox_offset=offset)
    keep = O.dropout_keep(x.numel(), p, seed, offset)
    _check(y.detach(), x.detach(), res.detach() if add else None, keep, p)
    grads = torch.autograd.grad(y, (x, res) if add else (x,), dy)
    _check(grads[0], dy, None, keep, p)
    if add:
        assert torch.equal(grads[1], dy)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("how", ["pitch", "odd_pitch", "shifted", "transposed", "permuted", "broadcast"])
def test_any_layout_gives_the_same_values(how, dt):
    from aotriton_b200 import autograd
    n, m = 48, 72
    base = torch.randn(n, m, device="cuda").to(dt)
    if how == "pitch":
        x = torch.empty(n, 96, device="cuda", dtype=dt)[:, :m]
    elif how == "odd_pitch":
        x = torch.empty(n, m + 5, device="cuda", dtype=dt)[:, 2:2 + m]
    elif how == "shifted":
        x = torch.empty(n * m + 1, device="cuda", dtype=dt)[1:].view(n, m)
    elif how == "transposed":
        x = torch.empty(m, n, device="cuda", dtype=dt).t()
    elif how == "permuted":
        x = torch.empty(8, m, 6, device="cuda", dtype=dt).permute(0, 2, 1)
        base = base.view(8, 6, m)
    else:
        base = base[:1].expand(n, m).contiguous()
        x = base[:1].expand(n, m)
    if how != "broadcast":
        x.copy_(base)
    want = autograd.dropout(base, 0.3, residual=base, philox_seed=9, philox_offset=4)
    assert torch.equal(autograd.dropout(x, 0.3, residual=base, philox_seed=9, philox_offset=4), want)
    assert torch.equal(autograd.dropout(base, 0.3, residual=x, philox_seed=9, philox_offset=4), want)
    assert torch.equal(autograd._Dropout.apply(x, x, 0.3, 9, 4), want)


def test_mask_is_the_attention_dropouts():
    """Element i of a row as wide as a score row has the bit that the attention's mask has there."""
    from aotriton_b200 import autograd, cabi
    rows, cols = 37, 132
    r = torch.empty(1, 1, rows, cols, device="cuda")
    assert cabi.debug_simulate_encoded_softmax(r, 0.4, torch.tensor([77], dtype=torch.uint64, device="cuda"), None, 1234) == 0
    y = autograd.dropout(torch.ones(rows, cols, device="cuda"), 0.4, philox_seed=77, philox_offset=1234)
    assert torch.equal(y != 0, r[0, 0] > 0)


def test_not_finite_where_dropped():
    from aotriton_b200 import autograd
    for dt, n in ((F16, 4096), (BF16, 1003), (F32, 77)):
        keep = O.dropout_keep(n, 0.5, 3, 8).cuda()
        x = torch.where(keep, torch.ones(n, device="cuda"), torch.tensor(float("nan"), device="cuda")).to(dt)
        x[~keep & (torch.arange(n, device="cuda") % 2 == 0)] = float("inf")
        y = autograd.dropout(x, 0.5, philox_seed=3, philox_offset=8)
        assert torch.equal(y, torch.where(keep, 2.0, 0.0).to(dt))


def test_seeds_in_tensors_are_read_at_replay():
    from aotriton_b200 import autograd
    x = torch.randn(100, 64, device="cuda", dtype=F16).requires_grad_()
    seed, offset = torch.tensor([5], device="cuda"), torch.tensor([1 << 40], device="cuda", dtype=torch.uint64)

    def step():
        y = autograd.dropout(x, 0.25, residual=x.detach(), philox_seed=seed, philox_offset=offset)
        return y.detach(), torch.autograd.grad(y, x, torch.ones_like(x))[0]

    plain = lambda s: autograd.dropout(x.detach(), 0.25, residual=x.detach(), philox_seed=s, philox_offset=1 << 40)
    assert torch.equal(step()[0], plain(5))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for s in (5, 6):
        seed.fill_(s)
        graph.replay()
        assert torch.equal(got[0], plain(s))
        assert torch.equal(got[1] != 0, O.dropout_keep(6400, 0.25, s, 1 << 40).view(100, 64).cuda())
    # changed between forward and backward, outside a graph: refused
    y = autograd.dropout(x, 0.25, philox_seed=seed, philox_offset=3)
    seed.add_(1)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, torch.ones_like(x))


def test_second_derivative_and_partial_gradients():
    from aotriton_b200 import autograd
    x, dy = torch.randn(5, 40, device="cuda").requires_grad_(), torch.randn(5, 40, device="cuda").requires_grad_()
    y = autograd.dropout(x, 0.3, philox_seed=2, philox_offset=7)
    dx, = torch.autograd.grad(y, x, dy, create_graph=True)
    d, = torch.autograd.grad(dx, dy, torch.ones_like(dy))
    assert torch.equal(d, autograd.dropout(torch.ones_like(dy), 0.3, philox_seed=2, philox_offset=7))
    # the residual alone, and a gradient that is an expanded scalar
    r = torch.randn(5, 40, device="cuda").requires_grad_()
    autograd.dropout(x.detach(), 0.3, residual=r).sum().backward()
    assert torch.equal(r.grad, torch.ones_like(r))
    autograd.dropout(x, 0.3, philox_seed=2, philox_offset=7).sum().backward()
    assert torch.equal(x.grad, d.detach())


def test_in_place_and_beside():
    from aotriton_b200 import cabi
    x = torch.randn(33, 70, device="cuda")
    want = torch.empty_like(x)
    assert cabi.dropout(x, want, 0.2, residual=x, philox_seed_value=4, philox_offset2=5) == 0
    store = torch.full((35, 80), 7.0, device="cuda")
    view = store[1:34, 3:73]
    view.copy_(x)
    assert cabi.dropout(view, view, 0.2, residual=x, philox_seed_value=4, philox_offset2=5) == 0
    assert torch.equal(view, want)
    view.fill_(7.0)
    assert bool((store == 7.0).all())


@pytest.mark.parametrize("cols", [4096, 4093])
def test_offsets_beyond_32_bits(cols):
    """More than 2^31 elements: the last rows, forward and backward."""
    from aotriton_b200 import autograd
    n, p, seed = (2 ** 31 // cols + 40) // 4 * 4, 0.3, 7
    x = torch.zeros(n, cols, device="cuda", dtype=BF16)
    x[-4:] = torch.randn(4, cols, device="cuda").to(BF16)
    x.requires_grad_()
    y = autograd.dropout(x, p, philox_seed=seed, philox_offset=0)
    first = (n - 4) * cols      # (a multiple of four: the rows start at a counter)
    keep = O.dropout_keep(4 * cols, p, seed, first // 4)
    _check(y.detach()[-4:], x.detach()[-4:], None, keep, p)
    dx, = torch.autograd.grad(y, x, x.detach())
    assert torch.equal(dx, y.detach())
