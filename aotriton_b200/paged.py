"""Serving from a cache in pages: the books (block tables and slot maps), the writing of new tokens, and attention of the last tokens of each
sequence over its pages.  The reference has none of these.

A cache is a (pages, page_size, heads, dim) tensor of any strides with unit innermost stride -- of (pages, heads, page_size, dim) storage its transpose(1, 2).
Sequence z's token n lies in slot n % page_size of page block_table[z, n // page_size].  A decoding step is

    step = block_tables(table, lengths, new_tokens, free_pages, page_size, total_tokens, taken)
    paged_write(k, v, k_cache, v_cache, step.slots)
    out = paged_attention(q, k_cache, v_cache, table, step.lengths)

with nothing read back to the host, so that it can be captured into a CUDA graph.  These operators have no gradients: training and prompts go by
autograd.attention, varlen_attention and latent_attention.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
import torch.autograd.forward_ad as forward_ad

from . import cabi
from .autograd import _FLOATS, _check, _native, _on_its_device, _unit_rows
from .flash import hipError_t


class BlockTables(NamedTuple):
    """What block_tables returns, all on the device."""
    slots: torch.Tensor         # (total_tokens,) int64: the slot of each new token, packed in order of sequence; -1: none
    cu_seqlens: torch.Tensor    # (batch + 1,) int32: running sums of the new tokens, as varlen_attention takes them
    lengths: torch.Tensor       # (batch,) int32: the sequences' lengths with the new tokens that had room in total_tokens
    taken: torch.Tensor         # (1,) int32: pages of the free list that are gone now; more than it has: there were too few


def _no_gradient(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad(), or on detached tensors")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode gradient")


def _int32(t, dim, device):
    return isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.dim() == dim and t.device == device and (t.numel() == 0 or t.shape[-1] == 1 or t.stride(-1) == 1)


def _whole(x, least):
    return type(x) is int and least <= x < 1 << 31


@torch._disable_dynamo
@_on_its_device
def _block_tables(block_table, lengths, new_tokens, free_pages, page_size, total_tokens, taken):
    device = block_table.device
    r = BlockTables(torch.empty([total_tokens], device=device, dtype=torch.int64), torch.empty([len(lengths) + 1], device=device, dtype=torch.int32),
                    torch.empty_like(lengths), torch.empty([1], device=device, dtype=torch.int32))
    stream = torch.cuda.current_stream(device).cuda_stream
    _check(hipError_t(cabi.block_tables(block_table, lengths, new_tokens, free_pages, page_size, *r, taken=taken, stream=stream)), "block_tables")
    torch.autograd.graph.increment_version(block_table)
    return r


def block_tables(block_table, lengths, new_tokens, free_pages, page_size, total_tokens, taken=None):
    """The books of one step: which page and slot each new token gets.  Returns a BlockTables; `block_table` is extended in place.

    block_table: (batch, width) int32, row z naming the pages of sequence z; lengths, new_tokens: (batch,) int32, tokens that it holds and tokens that it
    takes (0: none); free_pages: (n,) int32, pages to be taken, in order; taken: (1,) int32, how many of them are gone already (None: none).  Sequence z's
    first ceil(lengths[z] / page_size) entries are its own; the pages it needs beyond them are taken off the free list in order of sequence and position
    and entered into its row, the rest of which is left as it is.  Calling it again on the same arguments gives the same.

    total_tokens, a number, is the room for slots, at least the sum of new_tokens as a rule; slots behind that sum are -1.  Tokens beyond it get neither slot nor page,
    and `lengths` and `taken` do not count them (cu_seqlens does): a later step can take them.  Where the row is too short or the free list used up, tokens have the
    slot -1 (paged_write skips them) and count, and `taken` exceeds the length of the free list in the second case."""
    if not torch.compiler.is_compiling():
        r = _native.block_tables(block_table, lengths, new_tokens, free_pages, page_size, total_tokens, taken)
        if r is not None:
            return BlockTables._make(r)
    if not isinstance(block_table, torch.Tensor) or not block_table.is_cuda or not _int32(block_table, 2, block_table.device):
        raise ValueError("block_tables: the block table is a (batch, width) int32 CUDA tensor with rows of unit stride")
    device, batch = block_table.device, block_table.shape[0]
    if not all(_int32(t, 1, device) and t.shape[0] == batch for t in (lengths, new_tokens)):
        raise ValueError("block_tables: lengths and new_tokens are contiguous int32 tensors on the table's device, one entry a row of it")
    if not _int32(free_pages, 1, device) or (taken is not None and not (_int32(taken, 1, device) and taken.numel() == 1)):
        raise ValueError("block_tables: free_pages and taken are contiguous int32 tensors on the table's device, taken of one element")
    if batch > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError("block_tables: rows of the block table overlap")
    if not _whole(page_size, 1) or not _whole(total_tokens, 0):
        raise ValueError(f"block_tables: page_size {page_size} and total_tokens {total_tokens}: whole numbers, 1 or more and 0 or more")
    return _block_tables(block_table, lengths, new_tokens, free_pages, page_size, total_tokens, taken)


def _is_cache(t, like):
    return t.dim() == 4 and t.is_cuda and t.dtype == like.dtype and t.device == like.device and (t.shape[3] == 1 or t.stride(3) == 1)


@torch._disable_dynamo
@_on_its_device
def _paged_write(k, v, k_cache, v_cache, slots):
    stream = torch.cuda.current_stream(k.device).cuda_stream
    _check(hipError_t(cabi.paged_write(k, v, k_cache, v_cache, slots, stream=stream)), "paged_write")
    torch.autograd.graph.increment_version([t for t in (k_cache, v_cache) if t is not None])


def paged_write(k, v, k_cache, v_cache, slots):
    """Writes new tokens into a paged cache, in place: k_cache[slot // page_size, slot % page_size] = k[t], the same for v.

    k, v: (tokens, heads, dim) of any strides; caches (pages, page_size, heads, dim), of k's type; slots: (tokens,) int64, as block_tables gives them.  A slot outside
    the cache (-1) is skipped; the slots of a call differ from one another (of two tokens with one slot, parts of either may be left).  v and
    v_cache may be None, and their dim another than the keys': a latent cache of (pages, page_size, width) is written from a latent vector and
    its position columns with cache[:, :, None, :n] and cache[:, :, None, n:]."""
    if not torch.compiler.is_compiling() and _native.paged_write(k, v, k_cache, v_cache, slots):
        return
    if (v is None) != (v_cache is None):
        raise ValueError("paged_write: values and their cache come together")
    for x, cache in ((k, k_cache), (v, v_cache)):
        if x is None and x is v:
            continue
        if not x.is_cuda or x.dim() != 3 or x.dtype not in _FLOATS or x.dtype != k.dtype or x.device != k.device or x.shape[:2] != k.shape[:2]:
            raise ValueError("paged_write: k and v are (tokens, heads, dim) CUDA tensors of one device and type, fp32, fp16 or bf16")
        if not _is_cache(cache, k) or cache.shape[2:] != x.shape[1:] or cache.shape[:2] != k_cache.shape[:2] or 0 in cache.shape[1:]:
            raise ValueError("paged_write: the caches are (pages, page_size, heads, dim) tensors of k's device and type, with its heads and dim and unit innermost stride")
    if slots.dtype != torch.int64 or slots.dim() != 1 or slots.shape[0] != k.shape[0] or slots.device != k.device or (slots.numel() > 1 and slots.stride(0) != 1):
        raise ValueError("paged_write: slots is a contiguous int64 tensor on k's device, one entry a token")
    _no_gradient("paged_write", k, v, k_cache, v_cache)
    k, v = _unit_rows(k), None if v is None else _unit_rows(v)
    if k.shape[0] and k_cache.shape[0]:
        _paged_write(k, v, k_cache, v_cache, slots)


@torch._disable_dynamo
@_on_its_device
def _paged_attention(q, k_cache, v_cache, block_table, lengths, query_lengths, window, sinks, sm_scale, return_lse, what):
    b, hq, sq, _ = q.shape
    out = torch.empty((b, sq, hq, v_cache.shape[3]), device=q.device, dtype=q.dtype).transpose(1, 2)
    lse = torch.empty((b * hq, sq), device=q.device, dtype=torch.float32) if return_lse else None
    if out.numel():
        args = (q, k_cache, v_cache, block_table, lengths, out)
        kw = dict(sm_scale=sm_scale, window=window, sinks=sinks, query_lengths=query_lengths, lse=lse, stream=torch.cuda.current_stream(q.device).cuda_stream)
        need = cabi.paged_attn_workspace(*args, **kw)
        if need < 0:
            _check(hipError_t(-need), what)
        workspace = torch.empty([need], device=q.device, dtype=torch.float32) if need else None
        _check(hipError_t(cabi.paged_attn(*args, workspace=workspace, **kw)), what)
    return (out, lse) if return_lse else out


def _aligned(q):
    """q with a unit innermost stride and rows that start on 16 bytes where its type and head dim allow it: itself or a copy (a few rows, beside a cache)."""
    q = _unit_rows(q)
    per = 16 // q.itemsize
    if q.shape[-1] % per == 0 and (q.data_ptr() % 16 or any(n > 1 and s % per for n, s in zip(q.shape[:3], q.stride()))):
        q = q.clone(memory_format=torch.contiguous_format)
    return q


def _attend(q, k_cache, v_cache, block_table, lengths, query_lengths, window, sinks, sm_scale, return_lse, what):
    if q.dim() != 4 or q.dtype not in _FLOATS or not q.is_cuda:
        raise ValueError(f"{what}: q is a (batch, heads, tokens, head dim) CUDA tensor of fp32, fp16 or bf16")
    batch = q.shape[0]
    if not _int32(block_table, 2, q.device) or block_table.shape[0] != batch:
        raise ValueError(f"{what}: the block table is a (batch, width) int32 tensor on q's device with rows of unit stride")
    if not _int32(lengths, 1, q.device) or lengths.shape[0] != batch:
        raise ValueError(f"{what}: lengths is a contiguous int32 tensor on q's device, one entry a sequence")
    if query_lengths is not None and (not _int32(query_lengths, 1, q.device) or query_lengths.shape[0] != batch):
        raise ValueError(f"{what}: query_lengths is a contiguous int32 tensor on q's device, one entry a sequence")
    if window is not None and not (type(window) is int and window >= 1) or type(sinks) is not int or sinks < 0:
        raise ValueError(f"{what}: window {window} and sinks {sinks}: whole numbers, 1 or more (or None) and 0 or more")
    if not q.shape[1] or not k_cache.shape[2] or q.shape[1] % k_cache.shape[2]:
        raise ValueError(f"{what}: {q.shape[1]} query heads over {k_cache.shape[2]} heads of the cache")
    if not 1 <= q.shape[3] <= 1024 or not 1 <= v_cache.shape[3] <= 1024:
        raise ValueError(f"{what}: head dims from 1 to 1024 are supported")
    if not k_cache.shape[1]:
        raise ValueError(f"{what}: pages without slots")
    _no_gradient(what, q, k_cache, v_cache)
    window, sinks = 0 if window is None else min(window, 2 ** 31 - 1), min(sinks, 2 ** 31 - 1)
    return _paged_attention(_aligned(q), k_cache, v_cache, block_table, lengths, query_lengths, window, sinks, float(sm_scale), bool(return_lse), what)


def paged_attention(q, k_cache, v_cache, block_table, lengths, window=None, sinks=0, query_lengths=None, sm_scale=None, return_lse=False):
    """Attention of the last Sq tokens of each sequence over its pages.  q: (B, Hq, Sq, D) of any strides; caches (pages, page_size, Hk, D), fewer heads than q's
    for GQA; block_table: (B, width) int32; lengths: (B,) int32, keys of each sequence, the queries' own among them (block_tables' lengths
    of this step).  Query m stands at position P = lengths - Sq + m and sees the keys n <= P; with a window those with n > P - window
    or n < sinks, as in sink_attention.  query_lengths: (B,) int32, where sequences have fewer queries than Sq: theirs are the first of their rows, at
    P = lengths - query_lengths + m, and the other rows' output is zero.  Returns (B, Hq, Sq, Dv) and, if asked for, the log-sum-exp (B * Hq, Sq).

    Rows that see nothing give zeros (log-sum-exp +inf), positions below 0 among them.  Keys of pages outside the cache (table entries below 0, say) are seen by nobody;
    what slots hold that nobody sees, NaN included, does not matter.  The work is shared out on the device by the lengths, so that
    a batch of very different ones keeps the GPU busy.  The same inputs give the same bits.  No gradient.

    fp16 and bf16 with head dims up to 128 that are multiples of 8, 16-byte aligned caches, pages of a multiple of 8 slots and few queries are fastest."""
    sm_scale = q.shape[-1] ** -0.5 if sm_scale is None else sm_scale
    number = type(v_cache) is int      # (which the native route takes for a latent cache's value_dim)
    if not number and not torch.compiler.is_compiling():
        r = _native.paged_attention(q, k_cache, v_cache, block_table, lengths, query_lengths, window, sinks, sm_scale, return_lse)
        if r is not None:
            return r
    for t in (k_cache, v_cache):
        if number or not _is_cache(t, q) or t.shape[:3] != k_cache.shape[:3]:
            raise ValueError("paged_attention: the caches are (pages, page_size, heads, dim) tensors of q's device and type with unit innermost stride")
    if k_cache.shape[3] != q.shape[-1]:
        raise ValueError(f"paged_attention: head dims {q.shape[-1]} of q and {k_cache.shape[3]} of the keys")
    return _attend(q, k_cache, v_cache, block_table, lengths, query_lengths, window, sinks, sm_scale, return_lse, "paged_attention")


def paged_latent_attention(q, cache, block_table, lengths, value_dim, sm_scale, query_lengths=None, return_lse=False):
    """Latent attention in its absorbed form: all heads read one latent row a token, whose first value_dim columns are also the values.
    q: (B, H, Sq, width), each head's queries already multiplied by its key expansion, followed by their position columns; cache: (pages, page_size, width); the
    output (B, H, Sq, value_dim) is still to be multiplied by each head's value expansion.  sm_scale is that of the expanded form, the inverse root of a
    head's key width there (autograd.latent_attention computes the same from expanded keys and values, with gradients).  The rest as in paged_attention."""
    if not torch.compiler.is_compiling():
        r = _native.paged_attention(q, cache, value_dim, block_table, lengths, query_lengths, None, 0, sm_scale, return_lse)
        if r is not None:
            return r
    if cache.dim() != 3 or not _is_cache(cache[:, :, None], q) or cache.shape[2] != q.shape[-1]:
        raise ValueError("paged_latent_attention: the cache is a (pages, page_size, width) tensor of q's device, type and width with unit innermost stride")
    if type(value_dim) is not int or not 1 <= value_dim <= cache.shape[2]:
        raise ValueError(f"paged_latent_attention: value_dim {value_dim} of {cache.shape[2]} columns")
    cache = cache[:, :, None]
    return _attend(q, cache, cache[..., :value_dim], block_table, lengths, query_lengths, None, 0, sm_scale, return_lse, "paged_latent_attention")
