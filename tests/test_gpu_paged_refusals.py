"""GPU: calls that the native route must not take for others."""
import pytest
import torch

from _paged_reference import make
from aotriton_b200 import paged

pytestmark = pytest.mark.gpu


def test_a_number_for_the_values_is_no_latent_cache():
    q, cache, _, table, lens = make(2, 16, 1, 1, 576, 512, 16, [40, 7], torch.bfloat16, shared=True)
    paged.paged_latent_attention(q, cache[:, :, 0], table, lens, 512, 0.1)
    with pytest.raises(ValueError, match="paged_attention: the caches"):
        paged.paged_attention(q, cache[:, :, 0], 512, table, lens, sm_scale=0.1)
