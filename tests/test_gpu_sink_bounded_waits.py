"""Bounded waits that run out in the kernels of sink attention: the forward for head dims up to 128, the split-key forward, and the backward
whose keys are walked in chunks.

One copy is left out with a wait limit of about a million cycles.  The kernel must return, the status word must name it, further work
must be refused until the reset, and the next call must give what an undisturbed one gives.
"""
import pytest
import torch

from aotriton_b200 import cabi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what,D,Sq,Sk,drop,lo,hi", [("forward", 128, 700, 700, 1, 0x100, 0x1000), ("forward", 64, 256, 256, 1, 0x100, 0x1000),
                                                     ("one token", 128, 1, 2048, 1, 0x5000, 0x6000), ("backward", 128, 700, 700, 2, 0x1000, 0x5000)])
def test_runs_out_cleanly(what, D, Sq, Sk, drop, lo, hi):
    L = cabi.lib()
    q, k, v = (torch.randn(1, h, s, D, device="cuda").half() for h, s in ((4, Sq), (2, Sk), (2, Sk)))
    do, out, lse, delta = torch.randn_like(q), torch.empty_like(q), *(torch.empty(4, Sq, device="cuda") for _ in range(2))
    grads = [torch.empty_like(t) for t in (q, k, v)]
    args = (q, k, v, out, do, *grads, lse, delta, 100, 4)
    workspace = torch.empty(cabi.sink_attn_bwd_workspace(*args, sm_scale=0.1), device="cuda")

    def call():
        if what == "backward":
            return cabi.sink_attn_bwd(*args, workspace=workspace, sm_scale=0.1)
        return cabi.sink_attn_fwd(q, k, v, out, lse, 100, 4, sm_scale=0.1)

    stream = torch.cuda.current_stream().cuda_stream
    assert L.ab200_kernel_status(1) == 0
    results = grads if what == "backward" else [out, lse]
    assert cabi.sink_attn_fwd(q, k, v, out, lse, 100, 4, sm_scale=0.1) == 0
    assert call() == 0
    torch.cuda.synchronize()
    want = [t.clone() for t in results]
    L.ab200_debug_bounded_wait_test(drop, 1000)
    try:
        assert call() == 0
        assert call() == 0      # queued behind the first: starts after the failure and leaves at once
    finally:
        L.ab200_debug_bounded_wait_test(0, 0)
    assert L.ab200_stream_check(stream) == 719
    code = L.ab200_kernel_status(0)
    assert lo <= code < hi, hex(code)
    assert call() == 719
    assert L.ab200_kernel_status(1) == code
    assert L.ab200_stream_check(stream) == 0
    for t in results:
        t.fill_(float("nan"))
    assert call() == 0
    torch.cuda.synchronize()
    for a, b in zip(results, want):
        assert torch.equal(a, b)
