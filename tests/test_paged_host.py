"""CPU: the operators over a paged cache and keys that share columns, as far as they go without a GPU: refusals, struct layouts, the C entries'
host logic on a pretended device, the device that is current when they are called."""
import ctypes as C
import subprocess
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from aotriton_b200 import autograd, cabi, paged

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture
def fake():
    L = cabi.lib()
    L.ab200_debug_host_calls(1, -1, 0, 0)
    try:
        yield L
    finally:
        L.ab200_debug_host_calls(0, -1, 0, 0)


def test_struct_layouts(tmp_path):
    src = tmp_path / "layout.c"
    names = {"ab200_block_tables_args": (cabi.BlockTablesArgs, ["block_table", "num_free", "total_tokens", "taken_out"]),
             "ab200_paged_write_args": (cabi.PagedWriteArgs, ["num_pages", "k", "v_stride", "k_cache", "slots"]),
             "ab200_paged_attn_args": (cabi.PagedAttnArgs, ["sm_scale", "q", "v_cache", "block_table", "table_width", "lengths", "workspace_floats"]),
             "ab200_shared_columns_args": (cabi.SharedColumnsArgs, ["k", "shared", "joined"])}
    prints = "".join(f'printf("%zu ", sizeof({n}));' + "".join(f'printf("%zu ", offsetof({n}, {f}));' for f in fields) for n, (_, fields) in names.items())
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "aotriton_b200.h"\nint main(void) {' + prints + "return 0; }")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [x for cls, fields in names.values() for x in (C.sizeof(cls), *(getattr(cls, f).offset for f in fields))]


def _tables_args(**kw):
    a = cabi.BlockTablesArgs()
    a.batch, a.page_size, a.table_width, a.table_stride, a.num_free, a.total_tokens = 3, 16, 10, 10, 5, 100
    a.block_table, a.lengths, a.new_tokens, a.free_pages, a.slots, a.cu_seqlens, a.new_lengths, a.taken_out = (0x1000 * i for i in range(1, 9))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_block_tables_entry(fake):
    f, count = fake.ab200_block_tables, lambda: fake.ab200_debug_host_call_count(7)
    assert f(_tables_args(), None) == 0 and count() == 1
    assert f(_tables_args(total_tokens=0, slots=None), None) == 0 and count() == 2      # sums are still written
    assert f(_tables_args(batch=0, block_table=None, lengths=None, new_tokens=None, new_lengths=None), None) == 0 and count() == 3
    assert f(_tables_args(num_free=0, free_pages=None, taken=0x9000), None) == 0 and count() == 4
    assert f(_tables_args(table_width=0, block_table=None), None) == 0 and count() == 5
    for bad, code in ((dict(batch=-1), 1), (dict(page_size=0), 1), (dict(table_width=-1), 1), (dict(num_free=-1), 1), (dict(total_tokens=-1), 1), (dict(cu_seqlens=None), 1),
                      (dict(taken_out=None), 1), (dict(slots=None), 1), (dict(lengths=None), 1), (dict(new_tokens=None), 1), (dict(new_lengths=None), 1),
                      (dict(block_table=None), 1), (dict(free_pages=None), 1), (dict(table_stride=9), 1), (dict(total_tokens=1 << 31), 801)):
        assert f(_tables_args(**bad), None) == code, bad
    assert f(None, None) == 1 and count() == 5


def _write_args(**kw):
    a = cabi.PagedWriteArgs()
    a.dtype, a.num_heads, a.head_dim_k, a.head_dim_v, a.page_size, a.num_pages, a.tokens = cabi.DTYPE_BF16, 2, 64, 64, 16, 10, 20
    a.k, a.v, a.k_cache, a.v_cache, a.slots = (0x1000 * i for i in range(1, 6))
    a.k_stride[:] = a.v_stride[:] = (128, 64)
    a.k_cache_stride[:] = a.v_cache_stride[:] = (2048, 128, 64)
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


def test_paged_write_entry(fake):
    f, count = fake.ab200_paged_write, lambda: fake.ab200_debug_host_call_count(7)
    good = [dict(), dict(head_dim_v=0, v=None, v_cache=None), dict(head_dim_k=63), dict(k=0x1002), dict(k_stride=(131, 65)), dict(dtype=cabi.DTYPE_FP32, k=0x1004)]
    for kw in good:
        assert f(_write_args(**kw), None) == 0, kw
    assert count() == len(good)
    for kw in (dict(tokens=0, k=None), dict(num_pages=0, k_cache=None)):      # nothing to write, or nowhere
        assert f(_write_args(**kw), None) == 0 and count() == len(good)
    for bad, code in ((dict(num_heads=0), 1), (dict(head_dim_k=0), 1), (dict(head_dim_v=-1), 1), (dict(page_size=0), 1), (dict(num_pages=-1), 1), (dict(tokens=-1), 1),
                      (dict(dtype=0), 801), (dict(dtype=4), 801), (dict(k=None), 1), (dict(v=None), 1), (dict(k_cache=None), 1), (dict(v_cache=None), 1), (dict(slots=None), 1),
                      (dict(k=0x1001), 1), (dict(num_heads=1 << 20), 801), (dict(num_pages=1 << 62), 801)):
        assert f(_write_args(**bad), None) == code, bad
    assert f(None, None) == 1 and count() == len(good)


def _view(ptr, shape, stride=None):
    v = cabi.View4()
    v.ptr = ptr
    n = 1
    for i in reversed(range(4)):
        v.size[i], v.stride[i] = shape[i], stride[i] if stride else n
        n *= shape[i]
    return v


def _attn_args(dtype=cabi.DTYPE_BF16, B=4, Hq=8, Hk=2, Sq=1, D=128, Dv=128, page=16, pages=100, width=50, latent=False, **kw):
    a = cabi.PagedAttnArgs()
    a.dtype, a.batch, a.num_head_q, a.num_head_k, a.seqlen_q, a.head_dim_qk, a.head_dim_vo, a.page_size = dtype, B, Hq, Hk, Sq, D, Dv, page
    a.sm_scale = 0.1
    a.q, a.out = _view(0x10000, (B, Hq, Sq, D)), _view(0x20000, (B, Hq, Sq, Dv))
    a.k_cache, a.v_cache = _view(0x30000, (pages, page, Hk, D)), _view(0x40000, (pages, page, Hk, Dv))
    if latent:
        a.v_cache = _view(0x30000, (pages, page, Hk, Dv), tuple(a.k_cache.stride))
    a.block_table, a.table_stride, a.table_width, a.lengths = 0x50000, width, width, 0x60000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_paged_attention_entry(fake):
    f, size, count = fake.ab200_paged_attn, fake.ab200_paged_attn_workspace, lambda: fake.ab200_debug_host_call_count(7)

    def run(a, launches=2):
        need = size(a, None)
        assert need > 0 and need % 4 == 0
        before = count()
        for ptr, n in ((None, need), (0x70000, need - 1), (0x70004, need)):
            a.workspace, a.workspace_floats = ptr, n
            assert f(a, None) == 1 and count() == before
        a.workspace, a.workspace_floats = 0x70000, need
        assert f(a, None) == 0 and count() == before + launches
        return need

    for kw in (dict(), dict(Sq=4), dict(D=64, Dv=64), dict(D=80, Dv=80), dict(dtype=cabi.DTYPE_FP32), dict(dtype=cabi.DTYPE_FP16, page=7), dict(D=1024, Dv=1024), dict(D=5, Dv=3),
               dict(window=100, sinks=4), dict(Hq=64, Hk=1, Sq=9), dict(Hk=1, D=576, Dv=512, latent=True), dict(Hq=100, Hk=1, D=576, Dv=512, latent=True, Sq=2),
               dict(pages=0), dict(width=0, block_table=None), dict(lse=0x80000, query_lengths=0x90000)):
        run(_attn_args(**kw))
    # the workspace follows from the shape and the table's width, and stops growing with it
    assert size(_attn_args(width=1000), None) == size(_attn_args(width=100000), None)
    n = count()
    for kw in (dict(B=0), dict(Sq=0)):
        a = _attn_args(**kw)
        assert size(a, None) == 0 and f(a, None) == 0 and count() == n
    for bad, code in ((dict(batch=-1), 1), (dict(num_head_q=0), 1), (dict(num_head_k=0), 1), (dict(num_head_k=3), 1), (dict(seqlen_q=-1), 1), (dict(page_size=0), 1),
                      (dict(table_width=-1), 1), (dict(window=-1), 1), (dict(sinks=-1), 1), (dict(head_dim_qk=0), 1), (dict(head_dim_vo=0), 1), (dict(head_dim_qk=1025), 801),
                      (dict(head_dim_vo=1025), 801), (dict(dtype=0), 801), (dict(dtype=4), 801), (dict(page_size=8), 1), (dict(lengths=None), 1), (dict(block_table=None), 1),
                      (dict(q=cabi.View4()), 1), (dict(out=cabi.View4()), 1), (dict(k_cache=_view(None, (100, 16, 2, 128))), 1), (dict(v_cache=_view(0x40000, (99, 16, 2, 128))), 1),
                      (dict(v_cache=_view(0x40001, (100, 16, 2, 128))), 1), (dict(k_cache=_view(0x30000, (100, 16, 2, 128), (8192, 512, 256, 2))), 1)):
        a = _attn_args(**bad)
        assert size(a, None) == -code and f(a, None) == code, bad
    assert size(_attn_args(B=1 << 20, Hq=1 << 10, Hk=1, Sq=1 << 10), None) == -801
    assert size(_attn_args(B=1 << 16, Hq=128, Hk=128, width=1 << 27), None) == -801      # (more tiles than are counted)
    assert f(None, None) == 1 and size(None, None) == -1 and count() == n
    # an error on the way comes back, with nothing launched after it
    a = _attn_args()
    a.workspace, a.workspace_floats = 0x70000, size(a, None)
    for call, after, launches in ((7, 0, 1), (7, 1, 2), (5, 0, 0), (4, 0, 0)):
        fake.ab200_debug_host_calls(1, call, 98, after)
        assert f(a, None) == 98 and count() == launches, call


def test_shared_columns_entries(fake):
    join, add, count = fake.ab200_join_columns, fake.ab200_sum_columns, lambda: fake.ab200_debug_host_call_count(7)

    def args(B=2, H=3, S=5, dn=128, dr=64, **kw):
        a = cabi.SharedColumnsArgs()
        a.dtype, a.k, a.shared, a.joined = cabi.DTYPE_FP16, _view(0x1000, (B, H, S, dn)), _view(0x2000, (B, 1, S, dr)), _view(0x3000, (B, H, S, dn + dr))
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    assert join(args(), None) == 0 and add(args(), None) == 0 and count() == 2
    assert join(args(dn=3, dr=2), None) == 0 and add(args(k=cabi.View4()), None) == 0 and count() == 4
    for kw in (dict(B=0), dict(S=0)):
        assert join(args(**kw), None) == 0 and add(args(**kw), None) == 0 and count() == 4
    assert add(args(H=0), None) == 0 and count() == 5 and join(args(H=0), None) == 0 and count() == 5      # (a sum of nothing is still written)
    for bad, code in ((dict(dtype=0), 801), (dict(shared=_view(0x2000, (2, 2, 5, 64))), 1), (dict(shared=_view(0x2000, (2, 1, 4, 64))), 1), (dict(shared=_view(0x2001, (2, 1, 5, 64))), 1),
                      (dict(shared=_view(None, (2, 1, 5, 64))), 1), (dict(joined=_view(None, (2, 3, 5, 192))), 1), (dict(joined=_view(0x3000, (2, 3, 5, 192), (3840, 960, 384, 2))), 1),
                      (dict(shared=_view(0x2000, (2, 1, 5, 192))), 1)):
        assert join(args(**bad), None) == code and add(args(**bad), None) == code, bad
    for bad in (dict(k=_view(0x1000, (2, 3, 5, 127))), dict(k=_view(0x1000, (2, 2, 5, 128))), dict(k=cabi.View4())):
        assert join(args(**bad), None) == 1, bad
    assert join(None, None) == 1 and add(None, None) == 1 and count() == 5


def test_backward_of_joined_keys_entry(fake):
    f, size, count = fake.ab200_attn_bwd_shared, fake.ab200_attn_bwd_shared_workspace, lambda: fake.ab200_debug_host_call_count(7)

    def args(dtype=cabi.DTYPE_BF16, B=2, H=4, Hk=2, S=300, D=192, Dv=128, **kw):
        a = cabi.BwdArgs()
        p = a.prob
        p.dtype, p.batch, p.num_head_q, p.num_head_k, p.max_seqlen_q, p.max_seqlen_k, p.head_dim_qk, p.head_dim_vo, p.sm_scale = dtype, B, H, Hk, S, S, D, Dv, 0.1
        a.q, a.k, a.v, a.out, a.dout, a.dq, a.dk, a.dv = (_view(0x10000000 * (i + 1), (B, h, S, d)) for i, (h, d) in
                                                          enumerate(((H, D), (Hk, D), (Hk, Dv), (H, Dv), (H, Dv), (H, D), (Hk, D), (Hk, Dv))))
        a.lse, a.delta = 0xa0000000, 0xb0000000
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    for kw, columns, launches in ((dict(), 64, 4), (dict(D=96, Dv=64), 32, 4), (dict(D=256, Dv=256), 64, 5)):      # delta, dK and dV (256: apart), dQ, the sum
        a = args(**kw)
        shared = _view(0xc0000000, (2, 1, 300, columns))
        need = size(a, columns, None)
        assert need == 2 * 2 * 300 * columns
        n = count()
        for ptr, floats in ((None, need), (0x5000, need - 1), (0x5004, need)):
            assert f(a, columns, shared, ptr, floats, None) == 1
        assert count() == n and f(a, columns, shared, 0x5000, need, None) == 0 and count() == n + launches, kw
    for kw, columns in ((dict(dtype=cabi.DTYPE_FP32), 64), (dict(D=40, Dv=24), 6), (dict(D=13, Dv=10), 3)):      # from dK itself
        assert size(args(**kw), columns, None) == 0 and f(args(**kw), columns, _view(0xc0000000, (2, 1, 300, columns)), None, 0, None) == 0, kw
    n, good = count(), _view(0xc0000000, (2, 1, 300, 64))
    for columns, shared in ((0, good), (192, good), (-1, good), (32, good), (64, None), (64, _view(0xc0000000, (2, 2, 300, 64))), (64, _view(0xc0000000, (2, 1, 299, 64))),
                            (64, _view(None, (2, 1, 300, 64)))):
        assert f(args(), columns, shared, 0x5000, 1 << 30, None) == 1
    assert size(args(), 192, None) == -1 and size(None, 64, None) == -1 and count() == n


class T:
    """What the checks look at: they come before anything touches the device."""
    def __init__(self, *shape, dtype=torch.float16, cuda=True, device="cuda:0", unit=1, grad=False):
        self.shape, self.dtype, self.is_cuda, self.device, self.unit, self.requires_grad = torch.Size(shape), dtype, cuda, device, unit, grad

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def stride(self, i):
        return self.unit if i in (-1, len(self.shape) - 1) else 1 << 20

    def __getitem__(self, i):      # cache[:, :, None], or its first columns
        if i == (slice(None), slice(None), None):
            return T(*self.shape[:2], 1, *self.shape[2:], dtype=self.dtype, cuda=self.is_cuda, device=self.device, unit=self.unit)
        return T(*self.shape[:-1], i[-1].stop, dtype=self.dtype, cuda=self.is_cuda, device=self.device, unit=self.unit)


def _ints(*shape, device="cpu"):
    return torch.zeros(shape, dtype=torch.int32, device=device)


@pytest.mark.parametrize("change", [
    dict(q=T(2, 4, 1, 64, cuda=False)), dict(q=T(2, 4, 64)), dict(q=T(2, 4, 1, 64, dtype=torch.float64)), dict(q=T(2, 3, 1, 64, device="cpu")), dict(q=T(2, 0, 1, 64, device="cpu")),
    dict(q=T(2, 4, 1, 32, device="cpu")), dict(k=T(9, 16, 2, 64, dtype=torch.bfloat16)), dict(k=T(9, 16, 64)), dict(k=T(9, 16, 2, 64, unit=2)), dict(k=T(9, 16, 2, 64, device="cuda:1")),
    dict(v=T(9, 8, 2, 64)), dict(v=T(9, 16, 2, 1025)), dict(k=T(9, 0, 2, 64), v=T(9, 0, 2, 64)), dict(table=_ints(3, 5)), dict(table=_ints(2)), dict(table=_ints(2, 5).long()),
    dict(table=_ints(5, 2).t()), dict(lengths=_ints(3)), dict(lengths=_ints(2, 1)), dict(lengths=_ints(2).long()), dict(lengths=_ints(4)[::2]), dict(query_lengths=_ints(3)),
    dict(query_lengths=_ints(2).float()), dict(window=0), dict(window=-1), dict(window=2.0), dict(window=True), dict(sinks=-1), dict(sinks=None), dict(sinks=1.0),
])
def test_paged_attention_refusals(change):
    dev = "cpu"      # (the index tensors are real ones: everything else stands on their device)
    a = dict(q=T(2, 4, 1, 64, device=torch.device(dev)), k=T(9, 16, 2, 64, device=torch.device(dev)), v=T(9, 16, 2, 64, device=torch.device(dev)), table=_ints(2, 5), lengths=_ints(2))
    for k, v in change.items():
        if isinstance(v, T) and v.device != "cuda:1":
            v.device = torch.device(dev)
        a[k] = v
    with pytest.raises(ValueError):
        paged.paged_attention(a["q"], a["k"], a["v"], a["table"], a["lengths"], window=a.get("window"), sinks=a.get("sinks", 0), query_lengths=a.get("query_lengths"), sm_scale=1.0)


@pytest.mark.parametrize("change", [dict(cache=T(9, 16, 1, 576)), dict(cache=T(9, 16, 512)), dict(cache=T(9, 16, 576, dtype=torch.bfloat16)), dict(cache=T(9, 16, 576, unit=2)),
                                    dict(value_dim=0), dict(value_dim=577), dict(value_dim=512.0), dict(value_dim=True), dict(lengths=_ints(3))])
def test_paged_latent_attention_refusals(change):
    dev = torch.device("cpu")
    a = dict(q=T(2, 16, 1, 576, device=dev), cache=T(9, 16, 576, device=dev), lengths=_ints(2), value_dim=512) | change
    if isinstance(a["cache"], T):
        a["cache"].device = dev
    with pytest.raises(ValueError):
        paged.paged_latent_attention(a["q"], a["cache"], _ints(2, 5), a["lengths"], a["value_dim"], 0.1)


def test_gradients_are_refused():
    dev = torch.device("cpu")
    q, c = T(2, 4, 1, 64, device=dev, grad=True), T(9, 16, 2, 64, device=dev)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged.paged_attention(q, c, c, _ints(2, 5), _ints(2))


@pytest.mark.parametrize("change", [dict(v=None), dict(k=T(5, 2)), dict(k=T(5, 2, 64, cuda=False)), dict(k=T(5, 2, 64, dtype=torch.int32)), dict(v=T(5, 2, 64, dtype=torch.bfloat16)),
                                    dict(v=T(6, 2, 64)), dict(k_cache=T(9, 16, 2, 32)), dict(k_cache=T(9, 16, 1, 64)), dict(k_cache=T(9, 16, 2, 64, unit=2)), dict(v_cache=T(8, 16, 2, 64)),
                                    dict(k_cache=T(9, 0, 2, 64), v_cache=T(9, 0, 2, 64)), dict(slots=_ints(5)), dict(slots=torch.zeros(4, dtype=torch.int64)),
                                    dict(slots=torch.zeros(10, dtype=torch.int64)[::2]), dict(slots=torch.zeros(5, 1, dtype=torch.int64))])
def test_paged_write_refusals(change):
    dev = torch.device("cpu")
    a = dict(k=T(5, 2, 64), v=T(5, 2, 64), k_cache=T(9, 16, 2, 64), v_cache=T(9, 16, 2, 64), slots=torch.zeros(5, dtype=torch.int64)) | change
    for t in a.values():
        if isinstance(t, T):
            t.device = dev
    with pytest.raises(ValueError):
        paged.paged_write(a["k"], a["v"], a["k_cache"], a["v_cache"], a["slots"])


def test_block_tables_refusals():
    for table in (_ints(2, 5), None, [[1]]):      # not on a GPU, not a tensor
        with pytest.raises(ValueError):
            paged.block_tables(table, _ints(2), _ints(2), _ints(5), 16, 10)

    class Table(torch.Tensor):
        is_cuda = True

    table = _ints(2, 5).as_subclass(Table)
    good = dict(lengths=_ints(2), new_tokens=_ints(2), free_pages=_ints(5), page_size=16, total_tokens=10, taken=_ints(1))
    with pytest.raises(ValueError, match="overlap"):
        paged.block_tables(_ints(1, 5).as_subclass(Table).expand(2, 5), **good)
    for bad in (dict(lengths=_ints(3)), dict(lengths=_ints(2).long()), dict(new_tokens=_ints(2, 1)), dict(new_tokens=_ints(1)), dict(free_pages=_ints(5).float()), dict(free_pages=_ints(10)[::2]),
                dict(page_size=0), dict(page_size=16.0), dict(page_size=True), dict(total_tokens=-1), dict(total_tokens=1 << 31), dict(taken=_ints(2)), dict(taken=3), dict(lengths=None)):
        with pytest.raises(ValueError):
            paged.block_tables(table, **(good | bad))


@pytest.mark.parametrize("change", [dict(q=T(1, 4, 8, 191)), dict(q=T(1, 3, 8, 192)), dict(k=T(1, 2, 8, 0)), dict(k=T(1, 0, 8, 128)), dict(r=T(1, 2, 8, 64)), dict(r=T(1, 1, 7, 64)),
                                    dict(r=T(1, 1, 8, 0)), dict(r=T(2, 1, 8, 64)), dict(v=T(1, 2, 7, 128)), dict(v=T(1, 2, 8, 513)), dict(v=T(1, 2, 8, 0)), dict(v=T(1, 2, 128)),
                                    dict(k=T(1, 2, 8, 128, dtype=torch.bfloat16)), dict(q=T(1, 4, 8, 192, cuda=False)), dict(q=T(2, 4, 8, 192)),
                                    dict(q=T(1, 4, 8, 514), k=T(1, 2, 8, 450))])
def test_latent_attention_refusals(change):
    a = dict(q=T(1, 4, 8, 192), k=T(1, 2, 8, 128), r=T(1, 1, 8, 64), v=T(1, 2, 8, 128)) | change
    with pytest.raises(ValueError):
        autograd.latent_attention(a["q"], a["k"], a["r"], a["v"])


def test_they_run_on_their_tensors_device(monkeypatch):
    """A default stream's handle names no device: the tensors' own is made the current one."""
    current, seen = [None], []

    class Device:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            current.append(self.device)

        def __exit__(self, *exc):
            current.pop()

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=0))
    for name, result in (("block_tables", 0), ("paged_write", 0), ("paged_attn", 0), ("paged_attn_workspace", 8), ("shared_columns", 0), ("attn_fwd", 0), ("attn_bwd_shared", 0),
                         ("attn_bwd_shared_workspace", 8)):
        monkeypatch.setattr(cabi, name, lambda *a, name=name, result=result, **kw: (seen.append((name, current[-1])), result)[1])
    monkeypatch.setattr(paged, "_check", lambda err, what: None)
    monkeypatch.setattr(autograd, "_check", lambda err, what: None)
    monkeypatch.setattr(autograd._native, "note_bwd_family", lambda: None)
    here = torch.device("cpu")
    paged._block_tables(_ints(2, 5), _ints(2), _ints(2), _ints(5), 16, 10, None)
    k, cache = torch.zeros(5, 2, 8), torch.zeros(9, 16, 2, 8)
    paged._paged_write(k, None, cache, None, torch.zeros(5, dtype=torch.int64))
    paged._paged_attention(torch.zeros(2, 4, 1, 8), cache, cache, _ints(2, 5), _ints(2), None, 0, 0, 1.0, False, "x")
    q, k, r = torch.zeros(1, 2, 5, 12), torch.zeros(1, 2, 5, 8, requires_grad=True), torch.zeros(1, 1, 5, 4, requires_grad=True)
    autograd._LatentAttention.apply(q, k, r, k, None, None, 0, 0, 0, 0, 0, 1.0, False).sum().backward()
    assert seen == [(n, here) for n in ("block_tables", "paged_write", "paged_attn_workspace", "paged_attn", "shared_columns", "attn_fwd", "attn_bwd_shared_workspace",
                                        "attn_bwd_shared")]
