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
