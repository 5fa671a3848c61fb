"""Few queries against long caches where a CTA walks over many more tiles of keys than its ring has stages: stages of tiles with keys that nobody
sees, whose rows the kernel clears, are filled again by later copies."""
import ctypes as C

import pytest
import torch

from _sink_reference import check, reference

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("sinks", [1, 5, 70])
@pytest.mark.parametrize("B,Hq,Hk,Sq,D,window,plan", [      # plan: pieces of the keys, consumer warps, ring stages
    (40, 16, 4, 1, 128, 2000, (1, 4, 3)),
    (160, 4, 1, 4, 64, 2000, (1, 4, 6)),
    (90, 8, 2, 7, 128, 1500, (1, 4, 6)),       # two tiles of rows
    (20, 8, 2, 3, 128, 5000, (4, 4, 3)),       # a cluster shares the keys
    (1, 8, 2, 1, 128, 9000, (8, 8, 6)),
])
def test_hidden_keys_in_stages_that_are_filled_again(B, Hq, Hk, Sq, D, window, plan, sinks, dt):
    from aotriton_b200 import autograd, cabi
    Sk = window + 500
    g = torch.Generator(device="cuda").manual_seed(window + sinks)
    q, k, v = (torch.randn(B, h, s, D, generator=g, device="cuda").to(dt) for h, s in ((Hq, Sq), (Hk, Sk), (Hk, Sk)))
    a = cabi.make_fwd_args(q, k, v, torch.empty_like(q), None, sm_scale=1.0)      # (the cut goes by the tiles that are seen, here nearly all)
    n = cabi.lib().ab200_debug_split_keys(C.byref(a), None)
    assert (n & 0xff, n >> 8 & 0xff, n >> 16) == plan and window // 64 // plan[0] > 2 * plan[2]
    dirty_k, dirty_v = k.clone(), v.clone()
    hidden = slice(sinks, Sk - Sq - window + 1)
    dirty_k[:, :, hidden] = float("nan")
    dirty_v[:, :, hidden] = float("inf")
    out, lse = autograd.sink_attention(q, dirty_k, dirty_v, window, sinks, return_lse=True)
    clean, clean_lse = autograd.sink_attention(q, k, v, window, sinks, return_lse=True)
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)
    for z in range(0, B, 10):
        part = [t[z:z + 10] for t in (q, k, v)]
        values, bounds = reference(*part, window, sinks, D ** -0.5)
        check("out", out[z:z + 10], values, bounds)
        check("lse", lse.view(B, Hq, Sq)[z:z + 10], values, bounds)
    for _ in range(10):
        assert torch.equal(autograd.sink_attention(q, dirty_k, dirty_v, window, sinks), out)
    torch.cuda.synchronize()
    assert cabi.lib().ab200_kernel_status(0) == 0
