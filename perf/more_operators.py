"""Operators of serving from a paged cache, and of layers whose keys and values come from one latent vector a token, timed as a decoding
step, a prompt or a training step calls them:

  tables   block tables and slot maps from request lengths (`paged.block_tables`).  Sequence z holds `lengths[z]` tokens in pages of
           `page` slots and takes `new[z]` more.  Token i of them stands at position p = lengths[z] + i, in page p // page of its row; pages beyond
           the ceil(lengths[z] / page) that it has come from the free list, in order of sequence and position.
  write    keys and values of new tokens, or a latent vector's two parts, written to their slots (`paged.paged_write`).
  paged    attention of the last sq tokens of each sequence over its pages (`paged.paged_attention`).  Query m of a sequence of n keys stands at
           position P = m + n - sq and sees the keys j <= P with j > P - window or j < sinks.
  absorb   the same with one latent row a token for all heads, whose first `dv` columns are the values (`paged.paged_latent_attention`).
  expand   attention whose heads' keys are their own columns followed by columns that all heads share (`autograd.latent_attention`).

A case is a dict of plain values; `op` is one of the five, `train` True for forward and backward.  Plain forms are in single precision.
Inputs follow from the seed alone.
"""
import math
import random

import torch

own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- the cases ------------------------------------------------------------------------------------------------
def _named(name, c):
    return dict(c, name=name) if name else c


def _tables(name, b, page, held, new_lo, new_hi, lens):
    """Sequences with 0 to `held` tokens that take new_lo to new_hi more."""
    return _named(name, dict(op="tables", train=False, dtype="int", b=b, page=page, held=held, new_lo=new_lo, new_hi=new_hi, lens=lens))


def _write(name, dtype, tokens, page, pages, hk, d, dv, layout="nhd", skip=0):
    """`tokens` rows into a cache of pages * page slots; one head and dv > 0 beside d: two parts of one latent row.  skip: every
    skip-th token has no slot."""
    return _named(name, dict(op="write", train=False, dtype=dtype, tokens=tokens, page=page, pages=pages, hk=hk, d=d, dv=dv, layout=layout, skip=skip))


def _paged(name, dtype, b, hq, hk, sq, d, page, lo, hi, lens, window=0, sinks=0, layout="nhd"):
    return _named(name, dict(op="paged", train=False, dtype=dtype, b=b, hq=hq, hk=hk, sq=sq, d=d, dv=d, page=page, lo=lo, hi=hi, lens=lens, window=window,
                             sinks=sinks, layout=layout))


def _absorb(name, dtype, b, hq, sq, d, dv, page, lo, hi, lens):
    return _named(name, dict(op="absorb", train=False, dtype=dtype, b=b, hq=hq, hk=1, sq=sq, d=d, dv=dv, page=page, lo=lo, hi=hi, lens=lens, window=0,
                             sinks=0, layout="nhd"))


def _expand(name, train, dtype, b, h, s, dn, dr, dv, causal=True):
    return _named(name, dict(op="expand", train=train, dtype=dtype, b=b, h=h, s=s, dn=dn, dr=dr, dv=dv, causal=causal))


def listed():
    return [
        # a decoding step's bookkeeping: one token for each conversation of a batch
        _tables("tables_step", 48, 16, 6000, 1, 1, 1),
        # prompts that arrive beside running conversations, some of which rest
        _tables("tables_prompts", 300, 64, 4000, 0, 4000, 2),
        # a decoding step's keys and values
        _write("write_step", "bf16", 48, 16, 1000, 8, 128, 128),
        # prompts' latent rows, from two tensors, with padding among the tokens
        _write("write_latent_prompts", "fp16", 20011, 64, 400, 1, 512, 64, skip=7),
        # one token of one conversation: latency is all there is
        _paged("paged_one", "bf16", 1, 32, 8, 1, 128, 16, 1500, 1500, 3),
        # one token each of conversations of very different lengths
        _paged("paged_batch", "bf16", 64, 32, 8, 1, 128, 64, 100, 8192, 4),
        # four tokens that were guessed ahead, checked at once, by a model with a sliding window and first keys that stay visible
        _paged("paged_window_check", "fp16", 24, 16, 8, 4, 64, 32, 40, 6007, 5, window=2048, sinks=4, layout="hnd"),
        # a few very long conversations
        _paged("paged_long", "bf16", 4, 32, 8, 1, 128, 64, 90000, 131072, 6),
        # one token each of a few conversations, the heads of one device of several
        _absorb("absorb_few_heads", "bf16", 8, 16, 1, 576, 512, 64, 500, 6007, 7),
        # one token each of many conversations, all heads on one device
        _absorb("absorb_many_heads", "bf16", 32, 128, 1, 576, 512, 64, 500, 8192, 8),
        # single precision, odd sizes, as a reference run uses it
        _expand("expand_train_fp32", True, "fp32", 2, 8, 500, 64, 32, 64),
        # a decoder's training step
        _expand("expand_train", True, "bf16", 1, 32, 4096, 128, 64, 128),
    ]


def _log(rng, lo, hi):
    """A whole number from lo..hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    half = rng.choice(["bf16", "fp16"])
    while True:
        kind = rng.choice(["tables", "write", "latent_write", "paged", "paged", "paged", "paged_fp32", "absorb", "absorb", "absorb", "expand", "expand"])
        page = rng.choice([16, 16, 32, 64, 64, 128])
        lens = rng.randrange(1 << 20)
        if kind == "tables":
            lo = rng.choice([0, 1])
            c = _tables(None, _log(rng, 1, 1000), page, _log(rng, 16, 8000), lo, max(lo, _log(rng, 1, 8000) if rng.random() < 0.6 else 1), lens)
            if c["b"] * c["new_hi"] > 1500000:
                continue
        elif kind in ("write", "latent_write"):
            tokens = _log(rng, 1, 20000)
            pages = (tokens + tokens // 3) // page + 8
            if kind == "write":
                d = rng.choice([64, 80, 128, 128])
                c = _write(None, rng.choice([half, half, "fp32"]), tokens, page, pages, rng.choice([1, 2, 4, 8, 8]), d, d, rng.choice(["nhd", "hnd"]),
                           skip=rng.choice([0, 0, 5]))
            else:
                c = _write(None, half, tokens, page, pages, 1, rng.choice([256, 512, 512]), rng.choice([32, 64, 64]), skip=rng.choice([0, 0, 5]))
        elif kind in ("paged", "paged_fp32"):
            fp32 = kind == "paged_fp32"
            hq, hk = rng.choice([(8, 8), (16, 4), (32, 8), (32, 8), (32, 4), (64, 8), (12, 12), (16, 1)])
            hi = _log(rng, 20, 2000 if fp32 else 65536)
            c = _paged(None, "fp32" if fp32 else half, _log(rng, 1, 16 if fp32 else 100), hq, hk, rng.choice([1, 1, 1, 1, 2, 5]), rng.choice([64, 128, 128, 80]),
                       page, max(1, hi // rng.choice([1, 3, 50])), hi, lens, layout=rng.choice(["nhd", "hnd"]))
            if rng.random() < 0.3:
                c["window"], c["sinks"] = _log(rng, 16, 4096), rng.choice([0, 1, 4, 17])
            if c["b"] * c["hi"] * (c["hq"] * c["sq"] + 4 * c["hk"]) > (20000000 if fp32 else 30000000) * (1 if fp32 else 1):
                continue
        elif kind == "absorb":
            hi = _log(rng, 20, 32768)
            d, dv = rng.choice([(576, 512), (576, 512), (576, 512), (288, 256)])
            c = _absorb(None, half, _log(rng, 1, 64), rng.choice([8, 16, 16, 20, 32, 64, 128]), rng.choice([1, 1, 1, 2, 3]), d, dv, page,
                        max(1, hi // rng.choice([1, 3, 50])), hi, lens)
            if c["b"] * c["hi"] * (c["hq"] * c["sq"] + 4) > 35000000:
                continue
        else:
            dtype = rng.choice([half, half, half, "fp32"])
            dn, dr, dv = rng.choice([(128, 64, 128), (128, 64, 128), (64, 32, 64), (96, 32, 80)])
            s = _log(rng, 30, 700 if dtype == "fp32" else 4096)
            c = _expand(None, rng.random() < 0.7, dtype, _log(rng, 1, 4), rng.choice([4, 8, 12, 16, 32]), s, dn, dr, dv, rng.random() < 0.8)
            if dtype == "fp32" and dn > 96 or c["b"] * c["h"] * s * s > 32 * 4096 * 4096:
                continue
        if _plain_elements(c) <= _plain_elements(_LARGEST[c["op"]]):
            return c


def _lengths(c):
    r = random.Random(c["lens"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["b"])]


def _requests(c):
    """(tokens held, tokens new) of each sequence of a `tables` case."""
    r = random.Random(c["lens"])
    return [r.randint(0, c["held"]) for _ in range(c["b"])], [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["b"])]


def _plain_elements(c):
    """What the plain form of a case costs: tokens, cache entries, scores and gathered elements."""
    if c["op"] == "tables":
        return sum(_requests(c)[1]) + 10 * c["b"]
    if c["op"] == "write":
        return c["tokens"] * c["hk"] * (c["d"] + c["dv"])
    if c["op"] == "expand":
        return c["b"] * c["h"] * c["s"] * c["s"] * (4 if c["train"] else 1) * (c["dn"] + c["dr"])
    return c["b"] * c["hi"] * (c["hq"] * c["sq"] + c["hk"] * (c["d"] + c["dv"]))


_LARGEST = {c["op"]: c for c in sorted(listed(), key=_plain_elements)}
_LARGEST["write"] = _write("", "bf16", 20011, 64, 400, 8, 128, 128)


# ---- inputs ---------------------------------------------------------------------------------------------------
class State:
    pass


def _pages(n, page):
    return (n + page - 1) // page


def _cache(rand, c, pages, heads, width):
    """(pages, page, heads, width): slots' heads next to each other, or ("hnd") a head's slots."""
    if c["layout"] == "hnd":
        return rand(pages, heads, c["page"], width).transpose(1, 2)
    return rand(pages, c["page"], heads, width)


def prepare(case, seed):
    c, s = case, State()
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES.get(c["dtype"])

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt)

    def shuffled(n):
        return torch.randperm(n, generator=g, device="cuda").to(torch.int32)

    s.case = c
    if c["op"] == "tables":
        held, new = _requests(c)
        have, want = [_pages(n, c["page"]) for n in held], [_pages(n + m, c["page"]) for n, m in zip(held, new)]
        s.total = sum(new)
        order = shuffled(sum(want) + 5)
        s.table = torch.full((c["b"], max(want) + 3), -1, dtype=torch.int32, device="cuda")
        at = torch.tensor(have, device="cuda")
        inside = torch.arange(s.table.shape[1], device="cuda")[None] < at[:, None]
        s.table[inside] = order[:sum(have)]
        s.free = order[sum(have):].contiguous()
        s.lengths = torch.tensor(held, dtype=torch.int32, device="cuda")
        s.new = torch.tensor(new, dtype=torch.int32, device="cuda")
    elif c["op"] == "write":
        # projections' outputs: columns of a wider product, as a layer hands them over
        both = rand(c["tokens"], c["hk"] * (c["d"] + c["dv"]))
        s.k, s.v = (t.view(c["tokens"], c["hk"], -1) for t in both.split([c["hk"] * c["d"], c["hk"] * c["dv"]], dim=1))
        if c["d"] == c["dv"]:
            s.k_cache, s.v_cache = (_cache(rand, c, c["pages"], c["hk"], c["d"]) for _ in range(2))
        else:
            cache = rand(c["pages"], c["page"], 1, c["d"] + c["dv"])
            s.k_cache, s.v_cache = cache[..., :c["d"]], cache[..., c["d"]:]
        s.slots = torch.randperm(c["pages"] * c["page"], generator=g, device="cuda")[:c["tokens"]]
        if c["skip"]:
            s.slots[::c["skip"]] = -1
    elif c["op"] in ("paged", "absorb"):
        lens = _lengths(c)
        need = [_pages(n, c["page"]) for n in lens]
        pages = sum(need) + 3
        s.lens = lens
        s.lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s.table = torch.full((c["b"], max(need) + 1), -1, dtype=torch.int32, device="cuda")
        inside = torch.arange(s.table.shape[1], device="cuda")[None] < torch.tensor(need, device="cuda")[:, None]
        s.table[inside] = shuffled(pages)[:sum(need)]
        s.q = rand(c["b"], c["sq"], c["hq"], c["d"]).transpose(1, 2)
        if c["op"] == "paged":
            s.k_cache, s.v_cache = (_cache(rand, c, pages, c["hk"], c["d"]) for _ in range(2))
        else:
            s.cache = rand(pages, c["page"], c["d"])
    else:
        b, h, n = c["b"], c["h"], c["s"]
        # the expansion's output holds each head's key columns and values side by side
        s.q = rand(b, n, h, c["dn"] + c["dr"]).transpose(1, 2)
        kv = rand(b, n, h, c["dn"] + c["dv"]).transpose(1, 2)
        s.k, s.v = kv[..., :c["dn"]], kv[..., c["dn"]:]
        s.shared = rand(b, n, 1, c["dr"]).transpose(1, 2)
        s.dout = rand(b, n, h, c["dv"]).transpose(1, 2)
        s.inputs = (s.q, s.k, s.shared, s.v)
        if c["train"]:
            for t in s.inputs:
                t.requires_grad_()
    s.scale = (192 if c["op"] == "absorb" else c["dn"] + c["dr"] if c["op"] == "expand" else c.get("d", 1)) ** -0.5
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------
def _plain_tables(s):
    page, b = s.case["page"], s.case["b"]
    held, new = s.lengths.long(), s.new.long()
    total = held + new
    have, want = (held + page - 1) // page, (total + page - 1) // page
    ends = torch.cat([new.new_zeros(1), new.cumsum(0)])
    fresh = want - have
    start = fresh.cumsum(0) - fresh
    place = torch.arange(s.table.shape[1], device="cuda")[None]
    index = (start[:, None] + place - have[:, None]).clamp(0, s.free.numel() - 1)
    table = torch.where((place >= have[:, None]) & (place < want[:, None]), s.free.long()[index], s.table.long())
    t = torch.arange(s.total, device="cuda")
    z = torch.bucketize(t, ends[1:], right=True).clamp(max=b - 1)
    p = held[z] + t - ends[z]
    slots = table[z, p // page] * page + p % page
    return table.int(), slots, ends.int(), total.int(), fresh.sum().view(1).int()


def _plain_write(s):
    kept = s.slots >= 0
    page = s.case["page"]
    # (the tokens without a slot go to a row behind the cache's)
    slots = torch.where(kept, s.slots, s.case["pages"] * page)
    outs = []
    for x, cache in ((s.k, s.k_cache), (s.v, s.v_cache)):
        rows = torch.cat([cache.flatten(0, 1), cache.new_zeros(1, *cache.shape[2:])])
        rows[slots] = x
        outs.append(rows[:-1].view(cache.shape))
    return tuple(outs)


def _plain_paged(s):
    c = s.case
    group = c["hq"] // c["hk"]
    if c["op"] == "paged":
        kc, vc = s.k_cache, s.v_cache
    else:
        kc, vc = s.cache[:, :, None], s.cache[:, :, None, :c["dv"]]
    b, width = s.table.shape
    at = s.table.long().clamp(min=0)

    def rows(cache):      # (b, hk, keys, columns)
        return cache[at].float().flatten(1, 2).transpose(1, 2)

    n, m = torch.arange(width * c["page"], device="cuda"), torch.arange(c["sq"], device="cuda")
    here = (m[None] + s.lengths.long()[:, None] - c["sq"])[:, :, None]
    seen = (n <= here) & (n < s.lengths[:, None, None])
    if c["window"]:
        seen &= (n > here - c["window"]) | (n < c["sinks"])
    q = s.q.float().reshape(b, c["hk"], group, c["sq"], c["d"]).flatten(2, 3)
    p = (q @ rows(kc).transpose(-1, -2)).mul_(s.scale)
    p.masked_fill_(~seen[:, None, None].expand(b, c["hk"], group, -1, -1).flatten(2, 3), -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ rows(vc)) * torch.where(total > 0, 1 / total, 0.0)
    return out.view(b, c["hq"], c["sq"], c["dv"]).to(s.q.dtype)


def _plain_expand(s):
    c = s.case
    q, k, shared, v = (t.detach().float() for t in s.inputs)
    k = torch.cat([k, shared.expand(-1, c["h"], -1, -1)], -1)
    p = (q @ k.transpose(-1, -2)).mul_(s.scale)
    if c["causal"]:
        n = torch.arange(c["s"], device="cuda")
        p.masked_fill_(n[None] > n[:, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.mul_(1 / p.sum(-1, keepdim=True))
    out = p @ v
    result = out.to(s.q.dtype)
    if not c["train"]:
        return result
    do = s.dout.float()
    dv = p.transpose(-1, -2) @ do
    ds = (do @ v.transpose(-1, -2)).sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(s.scale)
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    dshared = dk[..., c["dn"]:].sum(1, keepdim=True)
    return tuple(t.to(s.q.dtype) for t in (result, dq, dk[..., :c["dn"]], dshared, dv))


# ---- one pass -------------------------------------------------------------------------------------------------
def _own(s):
    from aotriton_b200 import autograd, paged

    c = s.case
    if c["op"] == "tables":
        r = paged.block_tables(s.table, s.lengths, s.new, s.free, c["page"], s.total)
        return s.table, r.slots, r.cu_seqlens, r.lengths, r.taken
    if c["op"] == "write":
        paged.paged_write(s.k, s.v, s.k_cache, s.v_cache, s.slots)
        return s.k_cache, s.v_cache
    if c["op"] == "paged":
        return paged.paged_attention(s.q, s.k_cache, s.v_cache, s.table, s.lengths, window=c["window"] or None, sinks=c["sinks"])
    if c["op"] == "absorb":
        return paged.paged_latent_attention(s.q, s.cache, s.table, s.lengths, c["dv"], s.scale)
    if not c["train"]:
        with torch.no_grad():
            return autograd.latent_attention(s.q, s.k, s.shared, s.v, causal=c["causal"])
    out = autograd.latent_attention(s.q, s.k, s.shared, s.v, causal=c["causal"])
    return (out.detach(),) + torch.autograd.grad(out, s.inputs, s.dout)


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"tables": _plain_tables, "write": _plain_write, "paged": _plain_paged, "absorb": _plain_paged, "expand": _plain_expand}[state.case["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------
def _seen(sq, n, window, sinks):
    """(scores that are not masked, keys that some query sees) of one head."""
    pairs, first = 0, None
    for p in range(n - sq, n):
        if p >= 0:
            recent = max(p - window + 1, 0) if window else 0
            pairs += p - recent + 1 + min(recent, sinks)
            first = recent if first is None else first
    return (pairs, n - first + min(first, sinks)) if first is not None else (0, 0)


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "tables":
        held, new = _requests(c)
        fresh = sum(_pages(n + m, c["page"]) - _pages(n, c["page"]) for n, m in zip(held, new))
        # slots written; free pages read and entered; lengths, new tokens, ends and sums
        return {"bytes": 8 * sum(new) + 8 * fresh + 16 * c["b"], "flops": 0}
    if c["op"] == "write":
        tokens = c["tokens"] - (-(-c["tokens"] // c["skip"]) if c["skip"] else 0)
        return {"bytes": 2 * size * tokens * c["hk"] * (c["d"] + c["dv"]) + 8 * c["tokens"], "flops": 0}
    if c["op"] == "expand":
        b, h, n, dk = c["b"], c["h"], c["s"], c["dn"] + c["dr"]
        pairs = b * h * (n * (n + 1) // 2 if c["causal"] else n * n)
        inputs = b * n * (h * (dk + c["dn"] + c["dv"]) + c["dr"])
        out = b * n * h * c["dv"]
        if not c["train"]:
            return {"bytes": size * (inputs + out), "flops": 2 * pairs * (dk + c["dv"])}
        return {"bytes": size * (2 * inputs + 2 * out), "flops": 2 * pairs * (4 * dk + 3 * c["dv"])}
    seen = [_seen(c["sq"], n, c["window"], c["sinks"]) for n in _lengths(c)]
    keys = sum(x[1] for x in seen)
    columns = c["hk"] * (c["d"] + c["dv"]) if c["op"] == "paged" else c["d"]
    return {"bytes": size * (keys * columns + c["b"] * c["hq"] * c["sq"] * (c["d"] + c["dv"])),
            "flops": 2 * c["hq"] * (c["d"] + c["dv"]) * sum(x[0] for x in seen)}


# ---- in 64 bits -----------------------------------------------------------------------------------------------
def _exact_paged(s):
    c = s.case
    table = s.table.cpu().tolist()
    out = torch.zeros(c["b"], c["hq"], c["sq"], c["dv"], dtype=torch.float64, device="cuda")
    for z, n in enumerate(s.lens):
        pages = torch.tensor(table[z][:-(-n // c["page"])], device="cuda")
        for h in range(c["hk"]):
            if c["op"] == "paged":
                k = s.k_cache[pages, :, h].reshape(-1, c["d"])[:n].double()
                v = s.v_cache[pages, :, h].reshape(-1, c["dv"])[:n].double()
            else:
                k = s.cache[pages].reshape(-1, c["d"])[:n].double()
                v = k[:, :c["dv"]]
            heads = slice(h * (c["hq"] // c["hk"]), (h + 1) * (c["hq"] // c["hk"]))
            for m in range(c["sq"]):
                p = n - c["sq"] + m      # this query's place
                if p < 0:
                    continue
                from_ = max(0, p + 1 - c["window"]) if c["window"] else 0
                first = min(c["sinks"], from_)
                kk, vv = (torch.cat([x[:first], x[from_:p + 1]]) for x in (k, v))
                x = s.q[z, heads, m].double() @ kk.T * s.scale
                e = torch.exp(x - x.max(dim=1, keepdim=True).values)
                out[z, heads, m] = e @ vv / e.sum(dim=1, keepdim=True)
    return out


def _exact_expand(s):
    c = s.case
    q, k, shared, v = (t.detach() for t in s.inputs)
    out = torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in s.inputs]
    dn = c["dn"]
    for z in range(c["b"]):
        r = shared[z, 0].double()
        for h in range(c["h"]):
            a, kk, vv = q[z, h].double(), k[z, h].double(), v[z, h].double()
            x = (a[:, :dn] @ kk.T + a[:, dn:] @ r.T) * s.scale
            if c["causal"]:
                x = x + torch.full_like(x, -math.inf).triu(1)
            w = torch.exp(x - torch.logsumexp(x, dim=1, keepdim=True))
            out[z, h] = o = w @ vv
            if c["train"]:
                g = s.dout[z, h].double()
                t = w * (g @ vv.T - (g * o).sum(dim=1, keepdim=True)) * s.scale
                grads[0][z, h] = torch.cat([t @ kk, t @ r], dim=1)
                grads[1][z, h] = t.T @ a[:, :dn]
                grads[2][z, 0] += t.T @ a[:, dn:]
                grads[3][z, h] = w.T @ g
    return (out, *grads) if c["train"] else out


def _exact_write(s):
    c = s.case
    source = torch.full((c["pages"] * c["page"],), -1, device="cuda")      # the token that each slot gets
    kept = s.slots >= 0
    source[s.slots[kept]] = torch.arange(c["tokens"], device="cuda")[kept]
    source = source.view(c["pages"], c["page"], 1, 1)
    return tuple(torch.where(source >= 0, x.double()[source[..., 0, 0].clamp(min=0)], cache.double()) for x, cache in ((s.k, s.k_cache), (s.v, s.v_cache)))


def exact(case, seed):
    if case["op"] == "tables":      # whole numbers: nothing to be off
        return None
    s = prepare(case, seed)
    return {"write": _exact_write, "expand": _exact_expand}.get(case["op"], _exact_paged)(s)
