"""GPU: attention over pages against its definition in 64 bits.  Every slot that nobody sees holds NaN."""
import pytest
import torch

from _paged_reference import check, make, reference
from aotriton_b200 import cabi, paged

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]
ALL = HALF + [torch.float32]


def run(b, hq, hk, sq, d, dv, page, lengths, dtype, window=None, sinks=0, query_lengths=None, **kw):
    q, kc, vc, table, lens = make(b, hq, hk, sq, d, dv, page, lengths, dtype, window=window, sinks=sinks, query_lengths=query_lengths, **kw)
    ql = None if query_lengths is None else torch.tensor(query_lengths, dtype=torch.int32, device="cuda")
    out, lse = paged.paged_attention(q, kc, vc, table, lens, window=window, sinks=sinks, query_lengths=ql, return_lse=True)
    want, want_lse, most = reference(q, kc, vc, table, lens, window, sinks, ql)
    check(out, want, most)
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty)
    assert ((lse.double() - want_lse)[~empty].abs() < 1e-3).all()
    assert cabi.lib().ab200_kernel_status(0) == 0
    return out, lse


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("page", [16, 64, 8, 24, 128, 1, 7])
def test_lengths_around_pages_and_tiles(dtype, page):
    lengths = [0, 1, page - 1, page, page + 1, 63, 64, 65, 130, 500]
    run(len(lengths), 8, 2, 1, 64, 64, page, lengths, dtype)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("d,dv", [(128, 128), (64, 64), (80, 80), (128, 64), (40, 72), (8, 8), (5, 3), (256, 256), (33, 300), (576, 512), (1024, 1024)])
def test_head_dims(dtype, d, dv):
    run(3, 4, 2, 1, d, dv, 16, [300, 77, 5], dtype)


@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 8), (12, 12), (16, 1), (32, 4), (40, 8), (64, 2), (20, 1), (96, 1)])
@pytest.mark.parametrize("sq", [1, 2, 5])
def test_groups(hq, hk, sq):
    run(2, hq, hk, sq, 128, 128, 32, [700, 129], torch.bfloat16)
    run(2, hq, hk, sq, 64, 64, 32, [1, 333], torch.float16)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 4), (64, 64), (100, 3), (128, 200), (500, 0), (2 ** 31 - 1, 5), (300, 130)])
def test_windows_and_first_keys(dtype, window, sinks):
    run(5, 8, 2, 3, 64, 64, 16, [1, 2, 100, 611, 1500], dtype, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", HALF)
def test_no_window_ignores_first_keys(dtype):
    q, kc, vc, table, lens = make(2, 4, 4, 1, 64, 64, 16, [50, 200], dtype)
    assert torch.equal(paged.paged_attention(q, kc, vc, table, lens), paged.paged_attention(q, kc, vc, table, lens, sinks=7))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_layouts_and_bad_pages(dtype, layout):
    run(6, 16, 4, 1, 128, 128, 16, [1, 40, 400, 17, 250, 1000], dtype, layout=layout, bad=2)
    run(3, 16, 4, 2, 64, 64, 8, [9, 300, 64], dtype, layout=layout, bad=3, seed=1)


@pytest.mark.parametrize("dtype", ALL)
def test_query_lengths_and_queries_before_the_first_key(dtype):
    run(6, 8, 4, 4, 64, 64, 16, [2, 100, 3, 50, 0, 700], dtype, query_lengths=[4, 0, 1, 3, 2, 4])
    run(3, 8, 4, 9, 128, 128, 16, [2, 9, 10], dtype)
    run(2, 8, 4, 3, 64, 64, 16, [90, 90], dtype, query_lengths=[-5, 99])


@pytest.mark.parametrize("sq", [16, 33, 70])
def test_many_queries(sq):
    run(2, 6, 2, sq, 128, 128, 16, [200, 71], torch.bfloat16, window=50, sinks=2)
    run(2, 6, 2, sq, 64, 64, 32, [200, 71], torch.float16)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("b", [1, 3, 50, 300])
def test_batches_of_very_different_lengths(dtype, b):
    lengths = [(37 * i * i + 11 * i) % 50 + (5000 if i % 17 == 3 else 0) for i in range(b)]
    run(b, 4, 1, 1, 64, 64, 16, lengths, dtype)


@pytest.mark.parametrize("dtype", ALL)
def test_two_streams_at_once(dtype):
    """Calls that overlap, each with a workspace of its own."""
    cases = [make(4, 8, 2, 1, 128, 128, 16, [1000, 3, 500, 2000], dtype, seed=i) for i in range(2)]
    want = [paged.paged_attention(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged.paged_attention(*cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_one_long_sequence():
    run(1, 8, 1, 1, 128, 128, 64, [40001], torch.bfloat16)
    run(1, 8, 1, 2, 64, 64, 16, [30000], torch.float16, window=20000, sinks=3)


@pytest.mark.parametrize("dtype", ALL)
def test_nothing_to_see(dtype):
    q, kc, vc, table, lens = make(2, 4, 2, 2, 64, 64, 16, [5, 20], dtype, poison=False)
    for args in ((q, kc, vc, table[:, :0], lens), (q, kc[:0], vc[:0], table, lens), (q, kc, vc, table, lens - 100)):
        out, lse = paged.paged_attention(*args, return_lse=True)
        assert (out == 0).all() and torch.isposinf(lse).all()
    assert paged.paged_attention(q[:0], kc, vc, table[:0], lens[:0]).shape == (0, 4, 2, 64)
    assert paged.paged_attention(q[:, :, :0], kc, vc, table, lens).shape == (2, 4, 0, 64)
    # lengths beyond the table are its width
    full = paged.paged_attention(q, kc, vc, table[:, :1], torch.full_like(lens, 16))
    assert torch.equal(paged.paged_attention(q, kc, vc, table[:, :1], torch.full_like(lens, 10 ** 9)), full)


@pytest.mark.parametrize("dtype", ALL)
def test_infinities_and_nan_in_sight(dtype):
    q, kc, vc, table, lens = make(2, 4, 2, 1, 64, 64, 16, [30, 200], dtype)
    page, slot = int(table[0, 1]), 3      # key 19 of sequence 0
    vc[page, slot, 0, 5] = float("nan")
    out = paged.paged_attention(q, kc, vc, table, lens)
    bad = torch.isnan(out)
    assert bad[0, :2, :, 5].all() and int(bad.sum()) == 2
    kc[page, slot, 1, :] = float("-inf")      # of the other head: scores of -inf or +inf, as the queries' signs have it; never of sequence 1
    out = paged.paged_attention(q, kc, vc, table, lens)
    assert not torch.isnan(out[1]).any()


@pytest.mark.parametrize("dtype", HALF)
def test_strides(dtype):
    q, kc, vc, table, lens = make(3, 8, 2, 2, 64, 64, 16, [33, 200, 150], dtype, poison=False)
    want = paged.paged_attention(q, kc, vc, table, lens)
    wide = torch.randn(*kc.shape[:2], 2, 200, device="cuda").to(dtype)
    for off in (0, 8, 3):      # (rows that start on 16 bytes, and rows that do not)
        kk, vv = wide[..., off:off + 64], wide[..., off + 72:off + 136]
        kk.copy_(kc), vv.copy_(vc)
        check(paged.paged_attention(q, kk, vv, table, lens), *reference(q, kc, vc, table, lens)[::2])
    assert torch.equal(paged.paged_attention(q.contiguous(), kc, vc, table, lens), want)
    turned = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(paged.paged_attention(turned, kc, vc, table, lens), want)
    odd = torch.empty(3, 8, 2, 67, device="cuda", dtype=dtype)[..., 3:].copy_(q)
    assert torch.equal(paged.paged_attention(odd, kc, vc, table, lens), want)


def test_a_cache_beyond_2_31_elements():
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB")
    pages, page, hk, d = 70000, 64, 4, 128      # 2.3e9 elements
    kc, vc = (torch.zeros(pages, page, hk, d, device="cuda", dtype=torch.float16) for _ in range(2))
    table = torch.tensor([[pages - 1, 0, pages - 2, 65536]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for p in table[0].tolist():
        kc[p], vc[p] = (torch.randn(page, hk, d, generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
    q = torch.randn(1, 8, 1, d, generator=g, device="cuda", dtype=torch.float16)
    lens = torch.tensor([250], dtype=torch.int32, device="cuda")
    out = paged.paged_attention(q, kc, vc, table, lens)
    small = [c[table[0].long()] for c in (kc, vc)]
    want, _, most = reference(q, *small, torch.arange(4, dtype=torch.int32, device="cuda")[None], lens)
    check(out, want, most)
    x = torch.randn(3, hk, d, generator=g, device="cuda", dtype=torch.float16)
    slots = torch.tensor([pages * page - 1, 0, -1], device="cuda")
    paged.paged_write(x, x, kc, vc, slots)
    assert torch.equal(kc[-1, -1], x[0]) and torch.equal(vc[0, 0], x[1])


@pytest.mark.parametrize("d", [128, 72, 5])
def test_the_same_bits_and_a_captured_call(d):
    q, kc, vc, table, lens = make(4, 8, 2, 1, d, d, 16, [1000, 3, 500, 4000], torch.bfloat16, spare=400)
    first = paged.paged_attention(q, kc, vc, table, lens)
    for _ in range(5):
        assert torch.equal(paged.paged_attention(q, kc, vc, table, lens), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged.paged_attention(q, kc, vc, table, lens)
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.paged_attention(q, kc, vc, table, lens)
    with torch.cuda.graph(other):
        out2 = paged.paged_attention(q, kc, vc, table, lens)
    lens.copy_(torch.tensor([10, 999, 16, 3500], dtype=torch.int32))      # shorter: other shares of the work
    want, _, most = reference(q, kc.nan_to_num(), vc.nan_to_num(), table, lens)
    kc.nan_to_num_(), vc.nan_to_num_()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        other.replay()
    graph.replay()
    torch.cuda.synchronize()
    check(out, want, most)
    assert torch.equal(out, out2)


def test_another_stream():
    q, kc, vc, table, lens = make(2, 8, 2, 1, 128, 128, 16, [1000, 300], torch.bfloat16)
    want = paged.paged_attention(q, kc, vc, table, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged.paged_attention(q, kc, vc, table, lens)
    side.synchronize()
    assert torch.equal(got, want)


def test_refused_with_gradients():
    q, kc, vc, table, lens = make(1, 4, 2, 1, 64, 64, 16, [20], torch.float16)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged.paged_attention(q.requires_grad_(), kc, vc, table, lens)
    with torch.no_grad():
        paged.paged_attention(q, kc, vc, table, lens)
