"""CPU: the backward for joined keys on a pretended device: sizes for which its workspace would not do are refused."""
import pytest

from aotriton_b200 import cabi
from test_paged_host import _view, fake  # noqa: F401  (a fixture)


def _args(dtype, keys, batch, **prob):
    a = cabi.BwdArgs()
    p = a.prob
    p.dtype, p.batch, p.num_head_q, p.num_head_k, p.max_seqlen_q, p.max_seqlen_k, p.head_dim_qk, p.head_dim_vo, p.sm_scale = dtype, 2, 4, 2, 300, 300, 192, 128, 0.1
    a.q, a.k, a.v, a.out, a.dout, a.dq, a.dk, a.dv = (_view(0x10000000 * (i + 1), (batch, h, s, d)) for i, (h, s, d) in
                                                      enumerate(((4, 300, 192), (2, keys, 192), (2, keys, 128), (4, 300, 128), (4, 300, 128), (4, 300, 192), (2, keys, 192),
                                                                 (2, keys, 128))))
    a.lse, a.delta = 0xa0000000, 0xb0000000
    for k, v in prob.items():
        setattr(p, k, v)
    return a


@pytest.mark.parametrize("dtype", [cabi.DTYPE_BF16, cabi.DTYPE_FP32])
def test_tensors_smaller_than_the_problem_are_refused(fake, dtype):  # noqa: F811
    f, size, count = fake.ab200_attn_bwd_shared, fake.ab200_attn_bwd_shared_workspace, lambda: fake.ab200_debug_host_call_count(7)
    padded = dict(cu_seqlens_q=0x100, cu_seqlens_k=0x200, varlen_type=cabi.VARLEN_PADDED)
    packed = dict(padded, varlen_type=cabi.VARLEN_COMPACT)
    for keys, batch, prob, good in ((300, 2, {}, True), (301, 3, {}, True), (299, 2, {}, False), (300, 1, {}, False), (300, 2, padded, True), (299, 2, padded, False),
                                    (300, 1, padded, False), (600, 1, packed, True), (40, 1, packed, True), (40, 0, packed, False)):
        a, shared, n = _args(dtype, keys, batch, **prob), _view(0xc0000000, (batch, 1, keys, 64)), count()
        need = size(a, 64, None)
        code = f(a, 64, shared, 0x5000, 1 << 40, None)
        if good:
            assert need == (batch * 2 * keys * 64 if dtype == cabi.DTYPE_BF16 else 0) and code == 0 and count() > n, (keys, batch, prob)
        else:
            assert need == -1 and code == 1 and count() == n, (keys, batch, prob)
