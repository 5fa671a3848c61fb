"""CPU: how calls over pages are cut, on a pretended device; a refusal."""
import pytest
import torch

from aotriton_b200 import cabi, paged
from test_paged_host import T, _attn_args, _ints, fake  # noqa: F401  (a fixture)


@pytest.mark.parametrize("dtype", [cabi.DTYPE_FP32, cabi.DTYPE_BF16])
@pytest.mark.parametrize("dv,blocks", [(129, 3), (256, 3), (257, 2), (512, 2), (1024, 2)])
def test_the_general_kernel_is_cut_for_the_blocks_that_fit(fake, dtype, dv, blocks):  # noqa: F811
    """Two partial results of 8 rows for each CTA: as many as an SM holds of the kernel that takes the values' width."""
    need = fake.ab200_paged_attn_workspace(_attn_args(dtype=dtype, B=64, D=1000, Dv=dv, page=16, width=500), None)
    assert need == 2 * fake.ab200_multiprocessor_count(None) * blocks * -(-8 * (dv + 2) // 4) * 4


def test_tables_with_room_for_more_tiles_than_are_counted(fake):  # noqa: F811
    """Some sequences a launch (and a join each): 16 prompts of 8192 queries, 32:8 heads, over tables with room for a million tokens, and a decoding step over wider ones."""
    f, size, count = fake.ab200_paged_attn, fake.ab200_paged_attn_workspace, lambda: fake.ab200_debug_host_call_count(7)
    for kw, launches in ((dict(B=16, Hq=32, Hk=8, Sq=8192, width=65536), 3), (dict(B=2, Hq=32, Hk=8, Sq=8192, width=65536), 1), (dict(B=33, Hq=1, Hk=1, width=1 << 27), 2),
                         (dict(B=33, Hq=1, Hk=1, width=1 << 27, lse=0x80000, query_lengths=0x90000, dtype=cabi.DTYPE_FP32), 3),
                         (dict(B=70, Hq=16, Hk=1, D=576, Dv=512, latent=True, width=1 << 27), 2)):
        a, n = _attn_args(**kw), count()
        need = size(a, None)
        assert need > 0 and count() == n
        a.workspace, a.workspace_floats = 0x70000, need
        assert f(a, None) == 0 and count() == n + 2 * launches, kw
    a = _attn_args(B=33, Hq=1, Hk=1, width=1 << 27)
    a.workspace, a.workspace_floats = 0x70000, size(a, None)
    for after, launches in ((0, 1), (1, 2), (2, 3)):      # an error on the way comes back, with nothing launched after it
        fake.ab200_debug_host_calls(1, 7, 98, after)
        assert f(a, None) == 98 and count() == launches


def test_a_number_for_the_values_is_no_latent_cache():
    dev = torch.device("cpu")
    with pytest.raises(ValueError, match="paged_attention: the caches"):
        paged.paged_attention(T(2, 16, 1, 576, device=dev), T(9, 16, 576, device=dev), 512, _ints(2, 5), _ints(2))
