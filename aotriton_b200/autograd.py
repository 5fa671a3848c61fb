"""torch.autograd wrappers over the operator: what a framework's SDPA integration calls.

Follows the reference's test-side wrappers (ROCm/aotriton modules/flash/tests/
attn_torch_function.py:87-270 and varlen_attn_torch_function.py:38-206): the forward allocates O
and the fp32 logsumexp, owns the Philox seed/offset scalars when dropout is on and hands the
values it actually used to the backward; the backward allocates dQ/dK/dV(/dB) and a delta scratch.
"""
from __future__ import annotations

import ctypes
import functools
import operator
import warnings

import torch

from . import cabi, flash, load_torch_ops
from .flash import hipError_t

try:
    _native = load_torch_ops()
except ImportError as e:      # (built where torch was missing, had no CUDA or was another version)
    if torch.version.cuda is not None:
        warnings.warn(f"aotriton_b200: {e}; attention calls take the Python way, which costs the host more", RuntimeWarning)

    class _native:
        _family = 0

        @staticmethod
        def attend(*args):
            return None

        @staticmethod
        def sink_attend(*args):
            return None

        @staticmethod
        def relative_bias(*args):
            return None

        @staticmethod
        def dropout(*args):
            return None

        @staticmethod
        def set_python_backward(fn):
            pass

        @staticmethod
        def set_python_function(name, fn):
            pass

        @classmethod
        def note_bwd_family(cls):
            cls._family = int(cabi.lib().ab200_last_bwd_family())

        @classmethod
        def last_bwd_family(cls):
            return cls._family

DEFAULT_PHILOX_SEED = 0x1BF52
DEFAULT_PHILOX_OFFSET_1 = 0x1D4000
DEFAULT_PHILOX_OFFSET_2 = 0x000B42


def _check(err, what):
    if err != hipError_t.hipSuccess:
        raise RuntimeError(f"{what} failed: {err}")


def _on_its_device(fn):
    """fn with the device of its first tensor as the current one.  A default stream's handle is 0 on every device, and the library takes it for
    the current device's."""
    @functools.wraps(fn)
    def run(*args, **kw):
        with torch.cuda.device(next(t for t in args if isinstance(t, torch.Tensor)).device):
            return fn(*args, **kw)
    return run


# (torch.compiler.disable, with the three seconds of its import left to the first compiled call)
@torch._disable_dynamo
def _apply_untraced(function, *args):
    return function.apply(*args)


def _apply(function, *args):
    """function.apply(*args); a compiled caller's graph breaks here.  (Traced, the Functions fail at the current stream's handle.)"""
    return _apply_untraced(function, *args) if torch.compiler.is_compiling() else function.apply(*args)


# A null device scalar: no elements, so no address on any device.
_NULL_SCALAR = torch.empty([0], dtype=torch.uint64)
# The counter of a persistent kernel: the kernels bring their own.
_NULL_COUNTER = torch.empty([0], dtype=torch.int32)


def _device_u64(device, value):
    """One uint64 on the device.  Filled by a kernel on the current stream: torch.tensor(..., device=...) copies
    from pageable host memory and waits for the stream."""
    if type(value) is int and 0 <= value < 1 << 64:
        return torch.full([1], value - (value >> 63 << 64), device=device, dtype=torch.int64).view(torch.uint64)
    return torch.tensor([value], device=device, dtype=torch.uint64)


def _philox_tensors(device, dropout_p, seed, offset1):
    """(philox seed, philox offset) of a call as device scalars.  The offset is the whole of it (offset1 +
    offset2), so the backward takes both as they are with a second offset of 0."""
    if dropout_p <= 0.0:
        return _NULL_SCALAR, _NULL_SCALAR
    if type(offset1) is not int or not 0 <= offset1 < 1 << 64:
        offset1 = int(torch.tensor([offset1], dtype=torch.uint64).item())
    return _device_u64(device, seed), _device_u64(device, (offset1 + DEFAULT_PHILOX_OFFSET_2) % (1 << 64))


def __getattr__(name):
    # Kernel family of the most recent backward (the library keeps it per thread, and autograd runs
    # backward on a thread of its own): 1 = general, 2 = tcgen05, 0 = none yet.
    if name == "last_bwd_family":
        return _native.last_bwd_family()
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def _int64(x):
    return type(x) is int and -(1 << 63) <= x < 1 << 63


def _attend(q, k, v, b, cu_q, cu_k, max_q, max_k, sm_scale, dropout_p, causal, return_lse, seed, offset1, op):
    """The native route (csrc/torch_ops.cc): the result, or None where the call is not an ordinary one -- other tensors, modes
    or argument types, graph capture by torch.compile.  Those go by the Function or the operators below."""
    if torch.compiler.is_compiling():
        return None
    if op and not (_int64(seed) and _int64(offset1)):      # (the operators take both, used or not, as 64-bit signed numbers)
        return None
    ct, wl, wr = flash.translate_causal(causal)
    if type(offset1) is int and 0 <= offset1 < 1 << 64:
        offset1 = (offset1 + DEFAULT_PHILOX_OFFSET_2) % (1 << 64)
    elif dropout_p > 0.0:
        return None
    return _native.attend(q, k, v, b, cu_q, cu_k, max_q, max_k, sm_scale, dropout_p, ct, wl, wr, return_lse, seed, offset1, op)


@_on_its_device
def _backward(q, k, v, b, o, do, L, cu_q, cu_k, seed, offset1, offset2, sm_scale, dropout_p, causal, max_q, max_k):
    """(dq, dk, dv, dbias) of a dense or, with cumulative lengths, a token-packed call."""
    do = do if do.stride(-1) == 1 else do.contiguous()
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    db = torch.empty_like(b) if b is not None else None
    delta = torch.empty_like(L)
    if cu_q is None:
        _check(flash.attn_bwd(q, k, v, b, sm_scale, o, do, dq, dk, dv, db, None, L, flash.eager_delta(delta), dropout_p, seed, offset1,
                              offset2, causal), "attn_bwd")
    else:
        _check(flash.attn_bwd_varlen(q, k, v, cu_q, cu_k, max_q, max_k, None, None, None, sm_scale, o, do, dq, dk, dv, None, None, L,
                                     flash.eager_delta(delta), dropout_p, seed, offset1, offset2, causal, "compact"), "attn_bwd (varlen)")
    _native.note_bwd_family()
    return dq, dk, dv, db


def _native_backward(q, k, v, b, o, do, L, cu_q, cu_k, seed, offset, sm_scale, dropout_p, causal_type, wl, wr, max_q, max_k):
    """The backward of a native call whose gradient, saved tensors or modes are not ordinary ones (csrc/torch_ops.cc)."""
    causal = (wl, wr) if causal_type == flash.CausalType.WINDOWED else False
    return _backward(q, k, v, b, o, do, L, cu_q, cu_k, seed.view(torch.uint64) if seed is not None else _NULL_SCALAR, _NULL_SCALAR,
                     offset if seed is not None else 0, sm_scale, dropout_p, causal, max_q, max_k)


_native.set_python_backward(_native_backward)


class _Attention(torch.autograd.Function):
    @staticmethod
    @_on_its_device
    def forward(ctx, q, k, v, b, causal, sm_scale, dropout_p, return_lse=False,
                philox_seed=DEFAULT_PHILOX_SEED, philox_offset1=DEFAULT_PHILOX_OFFSET_1):
        o = torch.empty((q.shape[0], q.shape[1], q.shape[2], v.shape[3]), device=q.device, dtype=q.dtype)
        M = torch.empty((q.shape[0] * q.shape[1], q.shape[2]), device=q.device, dtype=torch.float32)
        seed, offset = _philox_tensors(q.device, dropout_p, philox_seed, philox_offset1)
        _check(flash.attn_fwd(q, k, v, b, sm_scale, M, o, dropout_p, seed, offset, 0, _NULL_SCALAR, _NULL_SCALAR,
                              None, causal, _NULL_COUNTER), "attn_fwd")
        ctx.save_for_backward(q, k, v, b, o, M)
        ctx.sm_scale, ctx.causal, ctx.dropout_p = sm_scale, causal, dropout_p
        ctx.philox_seed, ctx.philox_offset = seed, offset
        return (o, M) if return_lse else o

    @staticmethod
    def backward(ctx, do, *unused):
        q, k, v, b, o, L = ctx.saved_tensors
        dq, dk, dv, db = _backward(q, k, v, b, o, do, L, None, None, ctx.philox_seed, ctx.philox_offset, 0, ctx.sm_scale, ctx.dropout_p,
                                   ctx.causal, 0, 0)
        return dq, dk, dv, db, None, None, None, None, None, None


def attention(q, k, v, b=None, causal=False, sm_scale=None, dropout_p=0.0, return_lse=False,
              philox_seed=DEFAULT_PHILOX_SEED, philox_offset1=DEFAULT_PHILOX_OFFSET_1):
    """O = dropout(softmax(Q K^T * sm_scale + b, mask)) V for (B, H, S, D) tensors (any strides with
    unit innermost stride).  `causal` is a bool, a (left, right) window or a flash.CausalType."""
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else sm_scale
    r = _attend(q, k, v, b, None, None, 0, 0, sm_scale, dropout_p, causal, return_lse, philox_seed, philox_offset1, False)
    return r if r is not None else _apply(_Attention, q, k, v, b, causal, sm_scale, dropout_p, return_lse, philox_seed, philox_offset1)


class _VarlenAttention(torch.autograd.Function):
    @staticmethod
    @_on_its_device
    def forward(ctx, q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, causal, sm_scale,
                dropout_p, return_lse=False, philox_seed=DEFAULT_PHILOX_SEED,
                philox_offset1=DEFAULT_PHILOX_OFFSET_1):
        # q, k, v: (1, H, total_tokens, D) views of THD storage
        o = torch.empty((1, q.shape[2], q.shape[1], v.shape[3]), device=q.device, dtype=q.dtype).transpose(1, 2)
        M = torch.empty((q.shape[1], q.shape[2]), device=q.device, dtype=torch.float32)
        seed, offset = _philox_tensors(q.device, dropout_p, philox_seed, philox_offset1)
        _check(flash.attn_fwd_varlen(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, None, None,
                                     None, sm_scale, M, o, dropout_p, seed, offset, 0, _NULL_SCALAR, _NULL_SCALAR, None,
                                     causal, _NULL_COUNTER, "compact"), "attn_fwd (varlen)")
        ctx.save_for_backward(q, k, v, o, M, cu_seqlens_q, cu_seqlens_k)
        ctx.max_seqlens = (max_seqlen_q, max_seqlen_k)
        ctx.sm_scale, ctx.causal, ctx.dropout_p = sm_scale, causal, dropout_p
        ctx.philox_seed, ctx.philox_offset = seed, offset
        return (o, M) if return_lse else o

    @staticmethod
    def backward(ctx, do, *unused):
        q, k, v, o, L, cu_q, cu_k = ctx.saved_tensors
        dq, dk, dv, _ = _backward(q, k, v, None, o, do, L, cu_q, cu_k, ctx.philox_seed, ctx.philox_offset, 0, ctx.sm_scale, ctx.dropout_p,
                                  ctx.causal, *ctx.max_seqlens)
        return (dq, dk, dv) + (None,) * 10


def varlen_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, causal=False,
                     sm_scale=None, dropout_p=0.0, return_lse=False):
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else sm_scale
    r = _attend(q, k, v, None, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, sm_scale, dropout_p, causal, return_lse,
                DEFAULT_PHILOX_SEED, DEFAULT_PHILOX_OFFSET_1, False)
    return r if r is not None else _apply(_VarlenAttention, q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, causal,
                                  sm_scale, dropout_p, return_lse)


# ---------------------------------------------------------------------------------------------
# torch.library custom operators: the form in which a framework's SDPA dispatcher would register
# this library (the reference is wired into PyTorch the same way on ROCm, README.md:71-75; its own
# tests wrap the operator in autograd.Function, tests/attn_torch_function.py:87-270).  The ops are
# opaque to tracing (fake implementations give shapes and dtypes) and carry an autograd formula,
# so torch.compile and torch.export keep them as single nodes.
def _lse_rows(q):
    return q.shape[0] * q.shape[1], q.shape[2]


@torch.library.custom_op("aotriton_b200::attn_fwd", mutates_args=())
@_on_its_device
def op_attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, bias: torch.Tensor | None, sm_scale: float,
                dropout_p: float, causal_type: int, window_left: int, window_right: int, philox_seed: int,
                philox_offset1: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Returns (out, logsumexp, philox seed used, philox offset used)."""
    o = torch.empty((q.shape[0], q.shape[1], q.shape[2], v.shape[3]), device=q.device, dtype=q.dtype)
    M = torch.empty(_lse_rows(q), device=q.device, dtype=torch.float32)
    seed, offset = _philox_tensors(q.device, dropout_p, philox_seed, philox_offset1)
    causal = (window_left, window_right) if causal_type == flash.CausalType.WINDOWED else False
    _check(flash.attn_fwd(q, k, v, bias, sm_scale, M, o, dropout_p, seed, offset, 0, _NULL_SCALAR, _NULL_SCALAR, None,
                          causal, _NULL_COUNTER), "attn_fwd")
    if dropout_p <= 0.0:
        seed = torch.zeros([1], device=q.device, dtype=torch.uint64)
        offset = torch.zeros([1], device=q.device, dtype=torch.uint64)
    return o, M, seed, offset


@op_attn_fwd.register_fake
def _(q, k, v, bias, sm_scale, dropout_p, causal_type, window_left, window_right, philox_seed, philox_offset1):
    o = q.new_empty((q.shape[0], q.shape[1], q.shape[2], v.shape[3]))
    M = q.new_empty(_lse_rows(q), dtype=torch.float32)
    s = q.new_empty([1], dtype=torch.uint64)
    return o, M, s, q.new_empty([1], dtype=torch.uint64)


@torch.library.custom_op("aotriton_b200::attn_bwd", mutates_args=())
@_on_its_device
def op_attn_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, bias: torch.Tensor | None, out: torch.Tensor,
                dout: torch.Tensor, lse: torch.Tensor, philox_seed: torch.Tensor, philox_offset: torch.Tensor,
                sm_scale: float, dropout_p: float, causal_type: int, window_left: int, window_right: int,
                deterministic: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Returns (dq, dk, dv, dbias); dbias is an empty tensor when there is no bias."""
    dout = dout if dout.stride(-1) == 1 else dout.contiguous()
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    db = torch.empty_like(bias) if bias is not None else None
    causal = (window_left, window_right) if causal_type == flash.CausalType.WINDOWED else False
    opts = flash.attn_options()
    opts.deterministic = bool(deterministic)
    _check(flash.attn_bwd(q, k, v, bias, sm_scale, out, dout, dq, dk, dv, db, flash.lazy_dq_acc(dq), lse,
                          flash.lazy_delta(lse), dropout_p, philox_seed if dropout_p > 0 else _NULL_SCALAR,
                          philox_offset if dropout_p > 0 else _NULL_SCALAR, 0, causal, opts), "attn_bwd")
    _native.note_bwd_family()
    return dq, dk, dv, db if db is not None else q.new_empty([0])


@op_attn_bwd.register_fake
def _(q, k, v, bias, out, dout, lse, philox_seed, philox_offset, sm_scale, dropout_p, causal_type, window_left,
      window_right, deterministic):
    return (torch.empty_like(q), torch.empty_like(k), torch.empty_like(v),
            torch.empty_like(bias) if bias is not None else q.new_empty([0]))


def _op_setup_context(ctx, inputs, output):
    q, k, v, bias, sm_scale, dropout_p, causal_type, wl, wr, _, _ = inputs
    out, lse, seed_out, off_out = output
    ctx.save_for_backward(q, k, v, bias, out, lse, seed_out, off_out)
    ctx.args = (sm_scale, dropout_p, causal_type, wl, wr)


def _op_backward(ctx, dout, dlse, dseed, doff):
    q, k, v, bias, out, lse, seed_out, off_out = ctx.saved_tensors
    sm_scale, dropout_p, causal_type, wl, wr = ctx.args
    dq, dk, dv, db = op_attn_bwd(q, k, v, bias, out, dout, lse, seed_out, off_out, sm_scale, dropout_p, causal_type,
                                 wl, wr, torch.are_deterministic_algorithms_enabled())
    return dq, dk, dv, (db if bias is not None else None), None, None, None, None, None, None, None


op_attn_fwd.register_autograd(_op_backward, setup_context=_op_setup_context)


def scaled_dot_product_attention(query, key, value, attn_mask=None, dropout_p=0.0, is_causal=False, scale=None,
                                 enable_gqa=False, philox_seed=DEFAULT_PHILOX_SEED,
                                 philox_offset1=DEFAULT_PHILOX_OFFSET_1):
    """torch.nn.functional.scaled_dot_product_attention's signature over the custom operators.
    attn_mask must be a floating-point additive bias broadcastable to (B, Hq, Sq, Sk) or None (the
    operator has no boolean-mask input; the reference's kernels take an additive bias only, and only
    without causal masking, aot/_common.py:24-27)."""
    if attn_mask is not None:
        if attn_mask.dtype == torch.bool:
            raise ValueError("boolean attn_mask is not supported; pass an additive floating-point bias")
        if is_causal:
            raise ValueError("attn_mask together with is_causal is not supported by the operator")
        attn_mask = attn_mask.to(query.dtype).expand(query.shape[0], query.shape[1], query.shape[2], key.shape[2])
        if attn_mask.stride(-1) != 1:
            attn_mask = attn_mask.contiguous()
    if not enable_gqa and query.shape[1] != key.shape[1]:
        raise ValueError("query and key head counts differ; pass enable_gqa=True")
    scale = query.shape[-1] ** -0.5 if scale is None else scale
    r = _attend(query, key, value, attn_mask, None, None, 0, 0, float(scale), float(dropout_p), bool(is_causal), False, philox_seed,
                philox_offset1, True)
    if r is not None:
        return r
    ct, wl, wr = flash.translate_causal(bool(is_causal))
    return op_attn_fwd(query, key, value, attn_mask, float(scale), float(dropout_p), ct, wl, wr, philox_seed,
                       philox_offset1)[0]


# ---------------------------------------------------------------------------------------------
# What stands around attention in a layer.  The reference has neither.
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _launch(fn, device, args):
    """An entry point of the C-ABI on the device's current stream."""
    return fn(args, torch.cuda.current_stream(device).cuda_stream)


def _sink_problem(cu_q, cu_k, max_q, max_k, varlen, sm_scale):
    kw = dict(sm_scale=sm_scale)
    if varlen:
        kw.update(cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, max_seqlen_q=max_q, max_seqlen_k=max_k, varlen_type=varlen)
    return kw


def _unit_rows(t):
    """t with a unit innermost stride: itself or a copy.  A single column keeps any stride through contiguous()."""
    if t.stride(-1) != 1:
        t = t.squeeze(-1).unsqueeze(-1) if t.shape[-1] == 1 else t.contiguous()
    return t


class _SinkAttention(torch.autograd.Function):
    @staticmethod
    @_on_its_device
    def forward(ctx, q, k, v, cu_q, cu_k, max_q, max_k, window, sinks, sm_scale, return_lse, varlen):
        b, hq, sq, _ = q.shape
        packed = varlen == cabi.VARLEN_COMPACT
        if packed:      # (1, H, tokens, D) views of (tokens, H, D) storage
            o = torch.empty((1, sq, hq, v.shape[3]), device=q.device, dtype=q.dtype).transpose(1, 2)
        else:
            o = torch.empty((b, hq, sq, v.shape[3]), device=q.device, dtype=q.dtype)
        lse = torch.empty((hq, sq) if packed else (b * hq, sq), device=q.device, dtype=torch.float32)
        if not q.numel() or not k.numel() or not v.numel():      # nobody, or nothing to see
            o.zero_()
            lse.fill_(float("inf"))
        else:
            kw = _sink_problem(cu_q, cu_k, max_q, max_k, varlen, sm_scale)
            stream = torch.cuda.current_stream(q.device).cuda_stream
            _check(hipError_t(cabi.sink_attn_fwd(q, k, v, o, lse, window, sinks, stream=stream, **kw)), "sink_attn_fwd")
        ctx.save_for_backward(q, k, v, o, lse, cu_q, cu_k)
        ctx.args = (max_q, max_k, window, sinks, sm_scale, varlen)
        ctx.mark_non_differentiable(lse)
        return (o, lse) if return_lse else o

    @staticmethod
    def backward(ctx, do, *unused):
        q, k, v, o, lse, cu_q, cu_k = ctx.saved_tensors
        return _sink_grad(q, k, v, o, do, lse, cu_q, cu_k, *ctx.args) + (None,) * 9


class _SinkAttentionGrad(torch.autograd.Function):
    """(dq, dk, dv): an operator of its own, which knows that it has no derivative."""

    @staticmethod
    @_on_its_device
    def forward(ctx, q, k, v, o, do, lse, cu_q, cu_k, max_q, max_k, window, sinks, sm_scale, varlen):
        if not q.numel() or not k.numel() or not v.numel():
            return torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        do = _unit_rows(do)
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        delta = torch.empty_like(lse)
        kw = _sink_problem(cu_q, cu_k, max_q, max_k, varlen, sm_scale)
        args = (q, k, v, o, do, dq, dk, dv, lse, delta, window, sinks)
        stream = torch.cuda.current_stream(q.device).cuda_stream
        need = cabi.sink_attn_bwd_workspace(*args, stream=stream, **kw)
        if need < 0:
            _check(hipError_t(-need), "sink_attn_bwd")
        workspace = torch.empty([need], device=q.device, dtype=torch.float32) if need else None
        _check(hipError_t(cabi.sink_attn_bwd(*args, workspace=workspace, stream=stream, **kw)), "sink_attn_bwd")
        _native.note_bwd_family()
        return dq, dk, dv

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("sink_attention has no second derivative")


def _sink_grad(q, k, v, o, do, lse, cu_q, cu_k, *numbers):
    """The gradients, of a Python call or of a native one whose own gradient or modes are not ordinary ones (csrc/torch_ops.cc).

    A saved-tensor hook may have handed back anything; the kernels go by addresses and by the types and sizes that the gradient came with."""
    bad = [t for t in (q, k, v, o) if t.dim() != 4 or t.dtype != do.dtype or t.device != do.device]
    bad += [t for t in (cu_q, cu_k) if t is not None and (t.dtype != torch.int32 or t.device != do.device or t.shape != cu_q.shape or not t.is_contiguous())]
    if (bad or lse.dim() != 2 or lse.dtype != torch.float32 or lse.device != do.device or not lse.is_contiguous()
            or lse.numel() != q.shape[0] * q.shape[1] * q.shape[2] or not o.shape == do.shape == (*q.shape[:3], v.shape[3])
            or k.shape[:3] != v.shape[:3] or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3] or k.shape[1] and q.shape[1] % k.shape[1]):
        raise ValueError("sink_attention: what was saved for the backward came back with other types, sizes or devices")
    return _SinkAttentionGrad.apply(q, k, v, o, do, lse, cu_q, cu_k, *numbers)


_native.set_python_function("sink_attention", _sink_grad)


def _sink_attention(q, k, v, cu_q, cu_k, max_q, max_k, window, sinks, sm_scale, return_lse, varlen):
    if not torch.compiler.is_compiling():
        r = _native.sink_attend(q, k, v, cu_q, cu_k, max_q, max_k, window, sinks, sm_scale, return_lse, varlen)
        if r is not None:
            return r
    for t in (q, k, v):
        if t.dim() != 4 or t.dtype not in _FLOATS or not t.is_cuda or t.dtype != q.dtype or t.device != q.device:
            raise ValueError("sink_attention: q, k and v are (batch, heads, tokens, head dim) CUDA tensors of one device and type, fp32, fp16 or bf16")
    if type(window) is not int or type(sinks) is not int or window < 1 or sinks < 0:
        raise ValueError(f"sink_attention: window {window} and sinks {sinks}: whole numbers, 1 or more and 0 or more")
    if k.shape[0] != q.shape[0] or v.shape[:3] != k.shape[:3] or k.shape[3] != q.shape[3] or not k.shape[1] or q.shape[1] % k.shape[1]:
        raise ValueError(f"sink_attention: shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)} do not go together")
    if not 1 <= q.shape[3] <= 512 or not 1 <= v.shape[3] <= 512:
        raise ValueError("sink_attention: head dims from 1 to 512 are supported")
    if varlen:
        for t in (cu_q, cu_k):
            if t.dim() != 1 or t.numel() < 2 or t.numel() != cu_q.numel() or t.dtype != torch.int32 or t.device != q.device or t.stride(0) != 1:
                raise ValueError("sink_attention: the cumulative lengths are contiguous int32 tensors on q's device, one entry more than there are sequences")
        if varlen == cabi.VARLEN_COMPACT and q.shape[0] != 1:
            raise ValueError("sink_attention: packed tokens are (1, heads, tokens, head dim)")
        if varlen == cabi.VARLEN_PADDED and cu_q.numel() != q.shape[0] + 1:
            raise ValueError("sink_attention: a padded batch has one sequence for each entry of the batch axis")
        if not 0 <= max_q <= q.shape[2] or not 0 <= max_k <= k.shape[2]:
            raise ValueError(f"sink_attention: longest sequences {max_q} and {max_k} do not fit {q.shape[2]} and {k.shape[2]} tokens")
        max_q = q.shape[2] if varlen == cabi.VARLEN_PADDED else max(max_q, 1)
        max_k = max(max_k, 1)
    window, sinks = min(window, 2 ** 31 - 1), min(sinks, 2 ** 31 - 1)
    q, k, v = map(_unit_rows, (q, k, v))
    return _apply(_SinkAttention, q, k, v, cu_q, cu_k, max_q, max_k, window, sinks, float(sm_scale), bool(return_lse), varlen)


def sink_attention(q, k, v, window, sinks, sm_scale=None, return_lse=False):
    """Attention with a sliding window and `sinks` first keys that stay visible, for (B, H, S, D) tensors of any strides.  Query m of Sq
    stands at the key position P = m + Sk - Sq (queries are the last of the keys' positions: Sq = Sk in training, Sq = 1 for one token against a cache)
    and sees the keys n <= P with n > P - window or n < sinks.  A query that sees nothing gives zeros (log-sum-exp +inf).  GQA by fewer
    heads in k and v; no bias, no dropout.  Only keys that some query sees are read, whole blocks of them; of a cache's others, what they hold (NaN too) does
    not matter in fp16 and bf16 with head dims up to 256 that are multiples of 8.  The log-sum-exp has no gradient."""
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else sm_scale
    return _sink_attention(q, k, v, None, None, 0, 0, window, sinks, sm_scale, return_lse, 0)


def varlen_sink_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, window, sinks, sm_scale=None, return_lse=False,
                          varlen_type="compact"):
    """sink_attention over sequences of different lengths, each with its own positions.  varlen_type "compact": token-packed (1, H, tokens, D)
    tensors, as for varlen_attention.  "padded": (B, H, S, D) tensors, such as a batch of caches, sequence z having the first
    cu_seqlens[z + 1] - cu_seqlens[z] tokens of its row.  Of either, what lies behind the sequences is not looked at, output rows there are
    zero (log-sum-exp +inf) and gradients there are zero.  max_seqlen_q and _k are at least the longest lengths."""
    if varlen_type not in ("compact", "padded"):
        raise ValueError(f"varlen_sink_attention: varlen_type {varlen_type!r} is not \"compact\" or \"padded\"")
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else sm_scale
    return _sink_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, window, sinks, sm_scale, return_lse,
                           flash.IVARLEN_TYPE[varlen_type])


def relative_position_borders(buckets, max_distance):
    """The smallest distance of each bucket of one direction but the first, as a tuple of whole numbers: the first half of the buckets (e)
    has a distance each, bucket k beyond takes the distances from e * (max_distance / e) ** ((k - e) / (buckets - e)) on.  Compared in
    whole numbers: a logarithm in floating point puts distances next to a border on either side of it."""
    try:      # (as Python's own: other whole numbers overflow below, and whatever equals them would find their answer)
        return _borders(operator.index(buckets), operator.index(max_distance))
    except TypeError:
        raise ValueError(f"relative position buckets: {buckets!r} and {max_distance!r} are not whole numbers") from None


@functools.lru_cache(maxsize=None)
def _borders(buckets, max_distance):
    e = buckets // 2
    if buckets < 2 or max_distance <= e:
        raise ValueError(f"relative position buckets: {buckets} a direction up to distance {max_distance}: at least 2, and a distance above {e}, are needed")
    borders = list(range(1, e + 1))
    for k in range(e + 1, buckets):
        lo, hi = borders[-1], max_distance      # the smallest r with (r / e) ** (buckets - e) >= (max_distance / e) ** (k - e)
        most = e ** (buckets - k) * max_distance ** (k - e)
        while lo < hi:
            mid = (lo + hi) // 2
            if mid ** (buckets - e) >= most:
                hi = mid
            else:
                lo = mid + 1
        borders.append(lo)
    return tuple(borders)


@functools.lru_cache(maxsize=None)
def _borders_bytes(borders):
    return bytes((ctypes.c_int32 * len(borders))(*borders))


def _bias_rows(heads, sq, sk, dtype, device):
    """(1, heads, sq, sk) with rows of a multiple of 32 bytes, which the kernels that read and write it take 16 or 32 bytes at a time."""
    per = 32 // dtype.itemsize
    return torch.empty((1, heads, sq, (sk + per - 1) // per * per), device=device, dtype=dtype)[..., :sk]


class _RelativeBias(torch.autograd.Function):
    @staticmethod
    @_on_its_device
    def forward(ctx, table, sq, sk, batch, borders, bidirectional, query_offset, dtype):
        bias = _bias_rows(table.shape[1], sq, sk, dtype, table.device)
        if bias.numel():
            a = cabi.make_relative_bias_args(table, bias, borders, bidirectional=bidirectional, query_offset=query_offset)
            _check(hipError_t(_launch(cabi.lib().ab200_relative_bias_fwd, table.device, a)), "relative_bias_fwd")
        ctx.args = (borders, bidirectional, query_offset)
        ctx.like = (table.shape, table.dtype)
        return bias.expand(batch, -1, -1, -1)

    @staticmethod
    def backward(ctx, grad):
        return (_RelativeBiasGrad.apply(grad, *ctx.like, *ctx.args),) + (None,) * 7


class _RelativeBiasGrad(torch.autograd.Function):
    """The table's gradient; linear in its input, its own derivative is the bias again."""

    @staticmethod
    @_on_its_device
    def forward(ctx, grad, shape, dtype, borders, bidirectional, query_offset):
        table = torch.empty(shape, device=grad.device, dtype=dtype)
        ctx.args = (*grad.shape[2:], grad.shape[0], borders, bidirectional, query_offset, grad.dtype)
        if not grad.numel():
            return table.zero_()
        kw = dict(bidirectional=bidirectional, query_offset=query_offset)
        need = _launch(cabi.lib().ab200_relative_bias_workspace, grad.device, cabi.make_relative_bias_args(table, grad, borders, **kw))
        if need < 0:
            _check(hipError_t(-need), "relative_bias_bwd")
        workspace = torch.empty([need], device=grad.device, dtype=torch.float32)
        a = cabi.make_relative_bias_args(table, grad, borders, workspace=workspace, **kw)
        _check(hipError_t(_launch(cabi.lib().ab200_relative_bias_bwd, grad.device, a)), "relative_bias_bwd")
        return table

    @staticmethod
    def backward(ctx, grad):
        return (_RelativeBias.apply(grad, *ctx.args),) + (None,) * 5


def relative_position_bias(table, seqlen_q, seqlen_k, batch=1, max_distance=128, bidirectional=True, query_offset=0, dtype=None):
    """The additive bias of `attention` from a learned (buckets, heads) table: (batch, heads, seqlen_q, seqlen_k), the batch axis
    with stride 0, bias[b, h, m, n] = table[bucket(n - m - query_offset), h].

    Distances r have a bucket each up to half of a direction's buckets, and share the others evenly over their logarithm up to
    max_distance, beyond which all have the last (relative_position_borders).  Bidirectional: r = |n - m - query_offset|, keys after
    the query's position take the second half of the table (whose size is even); otherwise later keys count as distance 0.  query_offset is the position of
    query 0 among the keys: seqlen_k - 1 for the last token alone.  `dtype`: of the bias, the table's own where not given; fp32, fp16 or
    bf16 each.  The table's gradient is summed over the batch in fp32, in a fixed order."""
    if table.dim() != 2 or table.dtype not in _FLOATS or not table.is_cuda:
        raise ValueError("relative_position_bias: the table is a (buckets, heads) CUDA tensor of fp32, fp16 or bf16")
    dtype = table.dtype if dtype is None else dtype
    if dtype not in _FLOATS:
        raise ValueError(f"relative_position_bias: a bias of {dtype} is not supported")
    buckets = table.shape[0]
    if bidirectional:
        if buckets % 2:
            raise ValueError("relative_position_bias: two directions need an even number of buckets")
        buckets //= 2
    if min(seqlen_q, seqlen_k, batch) < 0 or table.shape[1] < 1:
        raise ValueError("relative_position_bias: negative sizes, or no heads")
    if buckets > 128:
        raise ValueError("relative_position_bias: at most 128 buckets a direction")
    if abs(query_offset) >= 1 << 31:
        raise ValueError("relative_position_bias: query_offset beyond 32 bits")
    borders = relative_position_borders(buckets, max_distance)
    if borders[-1] >= 1 << 31:
        raise ValueError(f"relative_position_bias: the last bucket starts at distance {borders[-1]}, beyond 32 bits")
    if not torch.compiler.is_compiling():
        r = _native.relative_bias(table, seqlen_q, seqlen_k, batch, _borders_bytes(borders), bool(bidirectional), query_offset, dtype)
        if r is not None:
            return r
    return _apply(_RelativeBias, table, seqlen_q, seqlen_k, batch, borders, bool(bidirectional), query_offset, dtype)


def _as_rows(t):
    """t as (rows, cols) with rows of unit stride: a view where its strides allow one, else a copy."""
    if t.dim() == 0:
        return t.view(1, 1)
    if t.is_contiguous():
        return t.view(-1, t.shape[-1]) if t.numel() else t.reshape(0, 1)
    try:
        rows = t.view(-1, t.shape[-1])
    except RuntimeError:
        rows = None
    return rows if rows is not None and (rows.stride(1) == 1 or rows.shape[1] == 1) else t.contiguous().view(-1, t.shape[-1])


class _Dropout(torch.autograd.Function):
    @staticmethod
    @_on_its_device
    def forward(ctx, x, residual, dropout_p, seed, offset):
        out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        tensors = [t if isinstance(t, torch.Tensor) else None for t in (seed, offset)]
        if x.numel():
            rows, to = _as_rows(x), _as_rows(out)
            add = None if residual is None else _as_rows(residual)
            numbers = [0 if isinstance(t, torch.Tensor) else t for t in (seed, offset)]
            stream = torch.cuda.current_stream(x.device).cuda_stream
            _check(hipError_t(cabi.dropout(rows, to, dropout_p, residual=add, philox_seed=tensors[0], philox_offset1=tensors[1],
                                           philox_seed_value=numbers[0], philox_offset2=numbers[1], stream=stream)), "dropout")
        ctx.save_for_backward(*tensors)      # (changed in place before the backward: refused there)
        ctx.numbers = (seed, offset)
        ctx.dropout_p = dropout_p
        ctx.residual = residual is not None
        return out

    @staticmethod
    def backward(ctx, grad):
        saved = [t if t is not None else n for t, n in zip(ctx.saved_tensors, ctx.numbers)]
        for x, what in zip(saved, ("philox_seed", "philox_offset")):      # (a saved-tensor hook may hand back anything)
            _philox_number(x, what, grad.device)
        dx = _Dropout.apply(grad, None, ctx.dropout_p, *saved) if ctx.needs_input_grad[0] else None
        return dx, grad if ctx.residual and ctx.needs_input_grad[1] else None, None, None, None


def _python_dropout(grad, dropout_p, seed, offset):
    """The gradient of a native call whose own gradient or modes are not ordinary ones (csrc/torch_ops.cc)."""
    return _Dropout.apply(grad, None, dropout_p, seed, offset)


def _python_relative_bias_grad(grad, buckets, heads, dtype, borders, bidirectional, query_offset):
    borders = tuple((ctypes.c_int32 * (len(borders) // 4)).from_buffer_copy(borders))
    return _RelativeBiasGrad.apply(grad, (buckets, heads), dtype, borders, bidirectional, query_offset)


_native.set_python_function("dropout", _python_dropout)
_native.set_python_function("relative_bias", _python_relative_bias_grad)


def _philox_number(x, what, device):
    if isinstance(x, torch.Tensor):
        if x.numel() != 1 or x.dtype not in (torch.int64, torch.uint64) or x.device != device:
            raise ValueError(f"dropout: {what} is a 64-bit number or a tensor of one on the device of x")
        return x
    if type(x) is not int or not 0 <= x < 1 << 64:
        raise ValueError(f"dropout: {what} is a number from 0 to 2**64 - 1, or a tensor of one")
    return x


def dropout(x, dropout_p, residual=None, philox_seed=DEFAULT_PHILOX_SEED, philox_offset=DEFAULT_PHILOX_OFFSET_1):
    """residual + dropout(x), for hidden states of any shape: element i in logical order is kept (and divided by 1 - dropout_p) or dropped by word
    (0, 2, 1, 3)[i % 4] of Philox counter philox_offset + i // 4, the attention's generator and threshold.  The mask is never stored: the backward
    draws it again.  dropout_p is taken in 32 bits, as the attention takes it.  A layer's calls take offsets at least x.numel() // 4 + 1 apart.

    Seed and offset are numbers, or 64-bit tensors of one element on x's device, which a captured call reads when it is replayed.  x and residual
    (the same shape and type: fp32, fp16 or bf16) need no particular strides, but what is not rows of unit stride is copied first.
    The output is contiguous."""
    if x.dtype not in _FLOATS or not x.is_cuda:
        raise ValueError("dropout: x is a CUDA tensor of fp32, fp16 or bf16")
    if not 0.0 <= dropout_p <= 1.0:
        raise ValueError(f"dropout: dropout_p is {dropout_p}, not a probability")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("dropout: the residual has another shape, type or device than x")
    if not torch.compiler.is_compiling():
        r = _native.dropout(x, residual, dropout_p, philox_seed, philox_offset)
        if r is not None:
            return r
    seed, offset = _philox_number(philox_seed, "philox_seed", x.device), _philox_number(philox_offset, "philox_offset", x.device)
    return _apply(_Dropout, x, residual, float(dropout_p), seed, offset)
