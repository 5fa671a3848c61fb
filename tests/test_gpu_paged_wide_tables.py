"""GPU: tables with room for more tiles than one launch counts: a few launches, each with some of the sequences."""
import pytest
import torch

from _paged_reference import check, reference
from aotriton_b200 import cabi, paged

pytestmark = pytest.mark.gpu
PAGE, WIDTH = 1 << 20, 2047      # a row has room for 2^31 keys


@pytest.mark.parametrize("dtype,kind", [(torch.bfloat16, "paged"), (torch.float16, "latent"), (torch.float32, "paged")])
@pytest.mark.parametrize("some_queries", [False, True])
def test_sequences_of_every_launch(dtype, kind, some_queries):
    b, hq, sq, d, dv = 70, 4, 2, (192 if kind == "latent" else 16), (128 if kind == "latent" else 16)
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = torch.full((2, PAGE, 1, d), float("nan"), device="cuda", dtype=dtype)      # (keys behind 3000 of a page are seen by nobody)
    cache[:, :3000] = torch.randn(2, 3000, 1, d, generator=g, device="cuda").to(dtype)
    values = cache[..., :dv] if kind == "latent" else cache.clone()
    lengths = torch.tensor([(i * 577) % 3000 if i % 7 else i % 3 for i in range(b)], dtype=torch.int32, device="cuda")
    table = torch.full((b, WIDTH), -1, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(b, device="cuda") % 2
    q = torch.randn(b, sq, hq, d, generator=g, device="cuda").to(dtype).transpose(1, 2)
    ql = torch.tensor([i % (sq + 1) for i in range(b)], dtype=torch.int32, device="cuda") if some_queries else None
    before = cabi.lib().ab200_launch_count()
    if kind == "latent":
        out, lse = paged.paged_latent_attention(q, cache[:, :, 0], table, lengths, dv, 0.1, query_lengths=ql, return_lse=True)
    else:
        out, lse = paged.paged_attention(q, cache, values, table, lengths, sm_scale=0.1, query_lengths=ql, return_lse=True)
    assert cabi.lib().ab200_launch_count() - before >= 4
    want, want_lse, most = reference(q, cache, values, table, lengths, query_lengths=ql, sm_scale=0.1)
    check(out, want, most)
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), empty) and ((lse.double() - want_lse)[~empty].abs() < 1e-3).all()
    # the same sequences over tables of one page
    small = table[:, :1].contiguous()
    if kind == "latent":
        alike = paged.paged_latent_attention(q, cache[:, :, 0], small, lengths, dv, 0.1, query_lengths=ql)
    else:
        alike = paged.paged_attention(q, cache, values, small, lengths, sm_scale=0.1, query_lengths=ql)
    check(alike, want, most)
