"""CPU: how calls over pages are cut, on a pretended device."""
import pytest

from aotriton_b200 import cabi
from test_paged_host import _attn_args, fake  # noqa: F401  (a fixture)


@pytest.mark.parametrize("dtype", [cabi.DTYPE_FP32, cabi.DTYPE_BF16])
@pytest.mark.parametrize("dv,blocks", [(129, 3), (256, 3), (257, 2), (512, 2), (1024, 2)])
def test_the_general_kernel_is_cut_for_the_blocks_that_fit(fake, dtype, dv, blocks):  # noqa: F811
    """Two partial results of 8 rows for each CTA: as many as an SM holds of the kernel that takes the values' width."""
    need = fake.ab200_paged_attn_workspace(_attn_args(dtype=dtype, B=64, D=1000, Dv=dv, page=16, width=500), None)
    assert need == 2 * fake.ab200_multiprocessor_count(None) * blocks * -(-8 * (dv + 2) // 4) * 4
