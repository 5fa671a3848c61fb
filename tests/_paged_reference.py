"""Attention over pages from its definition in 64 bits, with what a kernel may be off by, and cases whose unseen slots hold NaN."""
import math

import torch


def visible(n_keys, queries, window, sinks, device):
    """(queries, n_keys): query m stands at n_keys - queries + m."""
    pos = torch.arange(n_keys - queries, n_keys, device=device)[:, None]
    n = torch.arange(n_keys, device=device)[None]
    return (n <= pos) & ((n > pos - window) | (n < sinks)) if window else n <= pos


def gather(cache, row, n):
    """Keys 0..n-1 of a sequence: (n, heads, dim), and which of them lie in the cache."""
    page = cache.shape[1]
    i = torch.arange(n, device=cache.device)
    ids = row[(i // page).clamp(max=max(len(row) - 1, 0))].long() if len(row) else torch.full((n,), -1, device=cache.device)
    there = (ids >= 0) & (ids < cache.shape[0])
    if not cache.shape[0]:
        return cache.new_zeros(n, *cache.shape[2:]), there
    return torch.where(there[:, None, None], cache[ids.clamp(0, cache.shape[0] - 1), i % page], 0), there


def reference(q, k_cache, v_cache, table, lengths, window=None, sinks=0, query_lengths=None, sm_scale=None):
    """(out, lse, most): in 64 bits, and how far the output may be off in q's type.

    A kernel rounds the weights to the type once (half a step each: u of them times |v|), the output once, and forms scores of d products and their
    sum in 32 bits: a weight is off by twice the score's error.  Weights below the type's normal range (fp16) are off by half its smallest step."""
    b, hq, sq, d = q.shape
    hk, dv = k_cache.shape[2], v_cache.shape[3]
    scale = d ** -0.5 if sm_scale is None else sm_scale
    out = torch.zeros(b, hq, sq, dv, dtype=torch.float64, device=q.device)
    most = torch.zeros_like(out)
    lse = torch.full((b * hq, sq), math.inf, dtype=torch.float64, device=q.device)
    u = torch.finfo(q.dtype).eps / 2 if q.dtype != torch.float32 else 2.0 ** -22      # (32 bits: a few roundings of the running sums)
    for z in range(b):
        n = max(0, min(int(lengths[z]), table.shape[1] * k_cache.shape[1]))
        ql = sq if query_lengths is None else max(0, min(int(query_lengths[z]), sq))
        if not n or not ql:
            continue
        k, there = gather(k_cache, table[z], n)
        v, _ = gather(v_cache, table[z], n)
        ok = visible(n, ql, window, sinks, q.device) & there[None]
        anyone = ok.any(0)      # (what nobody sees may be NaN)
        k, v = (torch.where(anyone[:, None, None], t, 0).double() for t in (k, v))
        for h in range(hq):
            kh, vh, qh = k[:, h // (hq // hk)], v[:, h // (hq // hk)], q[z, h, :ql].double()
            x = (qh @ kh.T * scale).masked_fill(~ok, -math.inf)
            top = x.max(1, keepdim=True).values
            e = torch.exp(x - top.clamp(min=-1e300))
            s = e.sum(1, keepdim=True)
            some = s > 0
            p = e / torch.where(some, s, 1)
            out[z, h, :ql] = p @ vh
            lse[z * hq + h, :ql] = torch.where(some, top + torch.log(s), math.inf)[:, 0]
            score = (d + 8) * 2.0 ** -24 * scale * (qh.abs() @ kh.abs().T).masked_fill(~ok, 0).amax(1, keepdim=True) + (x.abs().masked_fill(~ok, 0).amax(1, keepdim=True) + 8) * 2.0 ** -23
            weighed = p @ vh.abs()
            small = 2.0 ** -25 * n / torch.where(some, s, 1) * vh.abs().amax() if q.dtype == torch.float16 else 0.0
            most[z, h, :ql] = u * (weighed + out[z, h, :ql].abs()) * 1.05 + 3 * score * weighed + small + n * 2.0 ** -24 * weighed
    return out, lse, most


def check(got, want, most, what=""):
    bad = ~((got.double() - want).abs() <= most + 1e-30)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[0].tolist(), float((got.double() - want).abs().nan_to_num(1e9).max()))


def make(b, hq, hk, sq, d, dv, page, lengths, dtype=torch.bfloat16, layout="nhd", window=None, sinks=0, query_lengths=None, bad=0, shared=False, spare=3, seed=0,
         poison=True, device="cuda"):
    """(q, k_cache, v_cache, table, lengths): pages in any order, entries behind a sequence's pages negative or far too large, `bad` of its entries too, and
    NaN in every slot that no query sees.  shared: the values are the keys' first columns."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pages, width = sum(need) + spare, max(need + [0]) + 2
    order = torch.randperm(pages, generator=g).int()
    junk = torch.tensor([-1, pages, 2 ** 31 - 1, -2 ** 31], dtype=torch.int64)
    table = junk[torch.randint(4, (b, width + 5), generator=g)].int()
    at = 0
    for z in range(b):
        table[z, :need[z]] = order[at:at + need[z]]
        at += need[z]
        for _ in range(bad):
            if need[z]:
                table[z, int(torch.randint(need[z], (1,), generator=g))] = junk[int(torch.randint(4, (1,), generator=g))].int()
    table = table[:, :width]

    def rand(*shape):
        return torch.randn(*shape, generator=g).to(dtype)

    def cache(width):
        return rand(pages, hk, page, width).transpose(1, 2) if layout == "hnd" else rand(pages, page, hk, width)

    k_cache, v_cache = cache(d), cache(dv)
    if poison:
        seen = torch.zeros(pages, page, dtype=torch.bool)
        for z, n in enumerate(lengths):
            ql = sq if query_lengths is None else max(0, min(query_lengths[z], sq))
            if not n or not ql:
                continue
            ok = visible(n, ql, window, sinks, "cpu").any(0)
            i = torch.arange(n)[ok]
            ids = table[z][i // page].long()
            here = (ids >= 0) & (ids < pages)
            seen[ids[here], (i % page)[here]] = True
        k_cache[~seen] = float("nan")
        v_cache[~seen] = float("nan")
    q = rand(b, sq, hq, d).transpose(1, 2)
    move = (lambda t: t.to(device)) if device != "cpu" else (lambda t: t)

    def put(t):      # (layouts survive)
        return torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=device).copy_(t)

    k_cache = put(k_cache)
    v_cache = k_cache[..., :dv] if shared else put(v_cache)
    table = torch.full((b, width + 5), -7, dtype=torch.int32, device=device)[:, :width].copy_(table)
    return put(q), k_cache, v_cache, table, torch.tensor(lengths, dtype=torch.int32, device=device)
