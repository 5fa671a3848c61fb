"""CPU: the operators around attention, as far as they go without a GPU: bucket borders, refusals, struct layouts, the C entries' host
logic on a pretended device."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

from aotriton_b200 import autograd, cabi
from oracle import layer as O

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def fake():
    L = cabi.lib()
    L.ab200_debug_host_calls(1, -1, 0, 0)
    try:
        yield L
    finally:
        L.ab200_debug_host_calls(0, -1, 0, 0)


@pytest.mark.parametrize("per", [2, 3, 8, 16, 32, 128])
@pytest.mark.parametrize("far", [2, 20, 64, 128, 1000, 32768])
def test_borders_against_the_definition(per, far):
    if far <= per // 2:
        with pytest.raises(ValueError):
            autograd.relative_position_borders(per, far)
        return
    borders = autograd.relative_position_borders(per, far)
    assert len(borders) == per - 1
    for r in sorted({x for b in borders for x in (b - 1, b, b + 1)} | {0, 1, far, far + 1, 10 ** 6}):
        assert sum(b <= r for b in borders) == O.bucket(-r, per, far, False), r


def test_a_border_that_a_logarithm_would_miss():
    # 16 buckets a direction, 128: distance 8 * 16 ** (1 / 2) = 32 exactly starts its bucket
    assert 32 in autograd.relative_position_borders(16, 128) and 16 in autograd.relative_position_borders(16, 128)


@pytest.mark.parametrize("change", [
    dict(table=torch.zeros(32, 4)),                                  # not on a GPU
    dict(buckets=31), dict(max_distance=8), dict(dtype=torch.float64), dict(query_offset=1 << 31),
    dict(seqlen_q=-1), dict(batch=-1), dict(buckets=512), dict(dim=3), dict(table_dtype=torch.float64),
])
def test_bias_refusals(change):
    class Table:      # (what the checks look at: they come before anything touches the device)
        def __init__(self, shape, dtype):
            self.shape, self.dtype, self.is_cuda = torch.Size(shape), dtype, True

        def dim(self):
            return len(self.shape)

    table = change.pop("table", None)
    if table is None:
        table = Table((change.pop("buckets", 32), 4) + (1,) * (change.pop("dim", 2) - 2), change.pop("table_dtype", torch.float32))
    args = dict(seqlen_q=5, seqlen_k=6) | change
    with pytest.raises(ValueError):
        autograd.relative_position_bias(table, **args)


@pytest.mark.parametrize("p,res,kw", [(0.1, None, {}), (-0.1, None, {}), (float("nan"), None, {}), (1.5, None, {})])
def test_dropout_refusals(p, res, kw):
    class X:
        dtype, is_cuda, shape, device = torch.float16, True, torch.Size((2, 3)), torch.device("cuda", 0)

    with pytest.raises(ValueError):
        autograd.dropout(torch.zeros(2, 3), p, residual=res, **kw)      # not on a GPU
    if not 0 <= p <= 1:
        with pytest.raises(ValueError):
            autograd.dropout(X, p)
    else:
        for bad in (torch.zeros(2, 3), torch.zeros(3, dtype=torch.float16), torch.zeros(2, 3, dtype=torch.float16)):
            with pytest.raises(ValueError):
                autograd.dropout(X, p, residual=bad)
        for seed in (-1, 1 << 64, 1.0, True, torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)):
            with pytest.raises(ValueError):
                autograd._philox_number(seed, "philox_seed", torch.device("cuda", 0))


def test_struct_layouts(tmp_path):
    src = tmp_path / "layout.c"
    src.write_text(r"""
#include <stdio.h>
#include <stddef.h>
#include "aotriton_b200.h"
int main(void) {
  printf("%zu %zu %zu %zu ", sizeof(ab200_relative_bias_args), offsetof(ab200_relative_bias_args, borders),
         offsetof(ab200_relative_bias_args, bias), offsetof(ab200_relative_bias_args, workspace_floats));
  printf("%zu %zu %zu\n", sizeof(ab200_dropout_args), offsetof(ab200_dropout_args, out_stride), offsetof(ab200_dropout_args, philox_offset2));
  return 0;
}
""")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    R, D = cabi.RelativeBiasArgs, cabi.DropoutArgs
    assert got == [C.sizeof(R), R.borders.offset, R.bias.offset, R.workspace_floats.offset, C.sizeof(D), D.out_stride.offset, D.philox_offset2.offset]


def _bias_args(B=1, H=4, Sq=10, Sk=20, borders=None, **kw):
    a = cabi.RelativeBiasArgs()
    borders = list(range(1, 16)) if borders is None else borders
    a.dtype, a.table_dtype, a.num_buckets, a.num_heads, a.bidirectional = cabi.DTYPE_BF16, cabi.DTYPE_FP32, 32, H, 1
    a.borders = (C.c_int32 * len(borders))(*borders)
    a.table = 0x1000
    a.table_stride[0], a.table_stride[1] = H, 1
    a.bias.ptr = 0x10000
    for i, (n, s) in enumerate(zip((B, H, Sq, Sk), (H * Sq * Sk, Sq * Sk, Sk, 1))):
        a.bias.size[i], a.bias.stride[i] = n, s
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_bias_entries_on_a_pretended_device(fake):
    fwd, bwd, size = fake.ab200_relative_bias_fwd, fake.ab200_relative_bias_bwd, fake.ab200_relative_bias_workspace
    assert fwd(_bias_args(), None) == 0 and fake.ab200_debug_host_call_count(7) == 1
    need = size(_bias_args(B=3), None)
    assert need > 0
    assert bwd(_bias_args(B=3), None) == 1      # no workspace
    assert bwd(_bias_args(B=3, workspace=0x5000, workspace_floats=need - 1), None) == 1
    assert fake.ab200_debug_host_call_count(7) == 1
    assert bwd(_bias_args(B=3, workspace=0x5000, workspace_floats=need), None) == 0 and fake.ab200_debug_host_call_count(7) == 3
    for bad, code in ((dict(num_buckets=31), 1), (dict(num_buckets=2), 1), (dict(num_buckets=0), 1), (dict(dtype=0), 801), (dict(dtype=9), 801),
                      (dict(table_dtype=0), 801), (dict(num_heads=0), 1), (dict(num_heads=3), 1), (dict(num_buckets=512), 801), (dict(table=None), 1),
                      (dict(borders=[0] + list(range(2, 16))), 1), (dict(borders=[2, 1] + list(range(3, 16))), 1), (dict(Sq=-1), 1), (dict(B=2), 1)):
        assert fwd(_bias_args(**bad), None) == code, bad
    assert fwd(None, None) == 1 and bwd(None, None) == 1 and size(None, None) == -1
    # nothing to do is done: no rows forward; backward the table's gradient is still written (zero)
    n = fake.ab200_debug_host_call_count(7)
    assert fwd(_bias_args(Sq=0), None) == 0 and fake.ab200_debug_host_call_count(7) == n
    assert bwd(_bias_args(Sq=0), None) == 0 and fake.ab200_debug_host_call_count(7) == n + 1
    fake.ab200_debug_host_calls(1, 7, 98, 0)
    assert fwd(_bias_args(), None) == 98


def _dropout_args(**kw):
    a = cabi.DropoutArgs()
    a.dtype, a.dropout_p, a.rows, a.cols = cabi.DTYPE_FP16, 0.1, 10, 16
    a.x, a.out, a.x_stride, a.out_stride = 0x1000, 0x2000, 16, 16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_dropout_entry_on_a_pretended_device(fake):
    f = fake.ab200_dropout
    count = lambda: fake.ab200_debug_host_call_count(7)
    assert f(_dropout_args(), None) == 0 and count() == 1
    assert f(_dropout_args(cols=15), None) == 0 and count() == 2      # rows that no vector divides: element by element
    assert f(_dropout_args(rows=1, cols=19), None) == 0 and count() == 4      # whole vectors, then the rest
    assert f(_dropout_args(rows=0), None) == 0 and f(_dropout_args(cols=0, x=None, out=None), None) == 0 and count() == 4
    for bad, code in ((dict(dropout_p=-0.5), 1), (dict(dropout_p=1.5), 1), (dict(dropout_p=float("nan")), 1), (dict(rows=-1), 1), (dict(x=None), 1),
                      (dict(out=None), 1), (dict(dtype=0), 801), (dict(rows=1 << 40, cols=1 << 40), 1), (dict(rows=1 << 30, cols=1 << 20), 801)):
        assert f(_dropout_args(**bad), None) == code, bad
    assert f(None, None) == 1 and count() == 4


def _attn_view(ptr, shape):
    v = cabi.View4()
    v.ptr = ptr
    for i, s in enumerate((shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3], 1)):
        v.size[i], v.stride[i] = shape[i], s
    return v


def _sink_args(cls, dtype=cabi.DTYPE_BF16, B=2, Hq=4, Hk=2, S=1024, D=128):
    a = cls()
    p = a.prob
    p.dtype, p.batch, p.num_head_q, p.num_head_k, p.max_seqlen_q, p.max_seqlen_k, p.head_dim_qk, p.head_dim_vo = dtype, B, Hq, Hk, S, S, D, D
    p.sm_scale = 1.0
    a.q, a.k, a.v, a.out = (_attn_view(0x10000000 * (i + 1), (B, h, S, D)) for i, h in enumerate((Hq, Hk, Hk, Hq)))
    a.lse = 0x50000000
    if cls is cabi.BwdArgs:
        a.dout, a.dq, a.dk, a.dv = (_attn_view(0x60000000 + 0x10000000 * i, (B, h, S, D)) for i, h in enumerate((Hq, Hq, Hk, Hk)))
        a.delta = 0xa0000000
    return a


def test_sink_entries_on_a_pretended_device(fake):
    fwd, bwd, size = fake.ab200_sink_attn_fwd, fake.ab200_sink_attn_bwd, fake.ab200_sink_attn_bwd_workspace
    count = lambda: fake.ab200_debug_host_call_count(7)
    a, b = _sink_args(cabi.FwdArgs), _sink_args(cabi.BwdArgs)
    assert fwd(a, 100, 4, None) == 0 and count() == 1 and fake.ab200_last_fwd_family() == 2
    need = size(b, 100, 4, None)
    assert need > 4 and size(b, 100, 0, None) == 4 and size(b, 1024, 4, None) == 4 and size(b, 2 ** 31 - 1, 2 ** 31 - 1, None) == 4
    for ptr, n in ((None, need), (0x5000, need - 1), (0x5004, need)):
        assert bwd(b, 100, 4, ptr, n, None) == 1 and count() == 1
    assert bwd(b, 100, 4, 0x5000, need, None) == 0 and count() == 5      # delta, dK/dV, the first keys' sums, dQ
    assert bwd(b, 100, 0, 0x5000, 4, None) == 0 and count() == 8
    assert fake.ab200_debug_host_call_count(6) == 0      # (the work counter is zeroed by the first launch)
    for window, sinks in ((0, 4), (-1, 4), (5, -1)):
        assert fwd(a, window, sinks, None) == 1 and bwd(b, window, sinks, 0x5000, need, None) == 1 and size(b, window, sinks, None) == -1
    for S in (0,):
        assert fwd(_sink_args(cabi.FwdArgs, S=S), 5, 1, None) == 1 and size(_sink_args(cabi.BwdArgs, S=S), 5, 1, None) == -1
    a.prob.dropout_p = b.prob.dropout_p = 0.1
    assert fwd(a, 5, 1, None) == 801 and size(b, 5, 1, None) == -801
    a.prob.dropout_p = b.prob.dropout_p = 0.0
    a.bias.ptr = 0x1000
    assert fwd(a, 5, 1, None) == 801
    # wide heads and single precision: for the first keys' partial sums alone
    for kw, d, launches in ((dict(D=256), 512, 5), (dict(dtype=cabi.DTYPE_FP32), 256, 3)):      # delta, the gradients (dV, dK, dQ or all), the sums
        b = _sink_args(cabi.BwdArgs, **kw)
        assert size(b, 100, 0, None) == 0 and size(b, 1000, 4, None) == 0
        items = size(b, 100, 4, None)
        assert items > 0 and items % (2 * 2 * 4 * d) == 0 and bwd(b, 100, 4, 0x5000, items - 1, None) == 1
        before = count()
        assert bwd(b, 100, 4, 0x5000, items, None) == 0 and count() == before + launches
    fake.ab200_debug_host_calls(1, 7, 98, 2)      # the third launch fails: nothing after it
    b = _sink_args(cabi.BwdArgs)
    assert bwd(b, 100, 4, 0x5000, need, None) == 98 and count() == 3


@pytest.mark.parametrize("change", [
    dict(window=0), dict(window=-3), dict(window=2.0), dict(window=True), dict(sinks=-1), dict(sinks=None), dict(heads=3), dict(kd=32), dict(vs=9), dict(kb=2),
    dict(d=513), dict(dtype=torch.float64), dict(vdtype=torch.bfloat16), dict(cpu=True),
])
def test_sink_refusals(change):
    class T:
        def __init__(self, shape, dtype):
            self.shape, self.dtype, self.is_cuda, self.device = torch.Size(shape), dtype, not change.get("cpu"), "cuda:0"

        def dim(self):
            return 4

        def stride(self, i):
            return 1

    dt, d = change.get("dtype", torch.float16), change.get("d", 64)
    q = T((1, 4, 8, d), dt)
    k = T((change.get("kb", 1), change.get("heads", 2), 8, change.get("kd", d)), dt)
    v = T((1, change.get("heads", 2), change.get("vs", 8), d), change.get("vdtype", dt))
    with pytest.raises(ValueError):
        autograd.sink_attention(q, k, v, change.get("window", 4), change.get("sinks", 1), sm_scale=1.0)


def test_varlen_sink_refusals():
    class T:
        def __init__(self, shape, dtype=torch.float16):
            self.shape, self.dtype, self.is_cuda, self.device = torch.Size(shape), dtype, True, torch.device("cpu")

        def dim(self):
            return 4

        def stride(self, i):
            return 1

    q, ends = T((2, 4, 8, 64)), torch.tensor([0, 8, 16], dtype=torch.int32)
    call = lambda q=q, a=ends, b=ends, mq=8, mk=8, how="padded": autograd.varlen_sink_attention(q, q, q, a, b, mq, mk, 4, 1, varlen_type=how)
    for bad in (dict(how="strided"), dict(how="compact"), dict(a=ends[:2]), dict(b=ends[:2]), dict(a=ends[:1], b=ends[:1]), dict(a=ends.long()), dict(mq=9), dict(mk=9),
                dict(mq=-1), dict(a=ends.view(1, 3)), dict(a=torch.zeros(6, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError):
            call(**bad)
