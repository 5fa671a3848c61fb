"""The operators that stand around attention in a layer, timed as a training step, a prompt or a decoding step calls them:

  sink     attention with a sliding window and a few first keys that stay visible (`autograd.sink_attention`,
           `autograd.varlen_sink_attention`).  Query m of a sequence of sq queries and sk keys stands at position
           P = m + sk - sq and sees the keys n <= P with n > P - window or n < sinks.
  bias     a learned relative position bias by buckets (`autograd.relative_position_bias`): out[b, h, m, n] =
           table[bucket(n - m - offset), h].  Distances r = |d| below half of a direction's `nb` buckets (e) have one each,
           those beyond share the others evenly over their logarithm, up to `far`:
           min(nb - 1, e + floor((nb - e) * log(r / e) / log(far / e))).  Both directions: nb is half of the table, keys behind the
           query's position take the second half; one: later keys count as distance 0.
  dropout  residual + keep(x) / (1 - p), the keep bits from Philox4x32-10 (`autograd.dropout`).  Element i of x in logical order takes word
           (0, 2, 1, 3)[i % 4] of counter offset + i / 4 and is kept where that word, as a signed number, is above the threshold
           trunc((p - 0.5) * 2^32) computed in single precision.

A case is a dict of plain values; `op` is one of the three, `train` True for forward and backward.  Plain forms are in single precision,
with sums along diagonals and distances in 64 bits.  Inputs follow from the seed alone.
"""
import math
import random

import numpy as np
import torch

own = False
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- the cases ------------------------------------------------------------------------------------------------
def _sink(name, api, train, dtype, b, hq, hk, sq, sk, d, window, sinks, layout="bhsd", lo=0, hi=0, lens=0):
    c = dict(op="sink", api=api, train=train, dtype=dtype, b=b, hq=hq, hk=hk, sq=sq, sk=sk, d=d, window=window, sinks=sinks, layout=layout, lo=lo,
             hi=hi, lens=lens)
    return dict(c, name=name) if name else c


def _bias(name, train, dtype, table, b, h, sq, sk, buckets, far, both, offset=0):
    c = dict(op="bias", train=train, dtype=dtype, table=table, b=b, h=h, sq=sq, sk=sk, buckets=buckets, far=far, both=both, offset=offset)
    return dict(c, name=name) if name else c


def _dropout(name, train, dtype, rows, cols, p, residual, pitch=0):
    c = dict(op="dropout", train=train, dtype=dtype, rows=rows, cols=cols, p=p, residual=residual, pitch=pitch or cols)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of one conversation that has outgrown its window: latency is all there is
        _sink("sink_step_one", "dense", False, "fp16", 1, 8, 8, 1, 1500, 64, 512, 4),
        # one token each of conversations of different lengths, over a batch of caches
        _sink("sink_step_batch", "padded", False, "bf16", 16, 32, 8, 1, 8192, 128, 2048, 4, layout="bshd", lo=100, hi=8192, lens=3),
        # prompts of different lengths, packed
        _sink("sink_prompts", "compact", False, "bf16", 12, 32, 8, 0, 0, 128, 512, 4, lo=32, hi=2048, lens=7),
        # single precision, odd sizes, as a reference run uses it
        _sink("sink_train_fp32", "dense", True, "fp32", 2, 8, 8, 500, 500, 64, 100, 3),
        # a decoder's training step on long sequences, grouped heads
        _sink("sink_train_long", "dense", True, "bf16", 1, 32, 8, 8192, 8192, 128, 1024, 4),
        # the bias of one decoding step
        _bias("bias_step", False, "bf16", "bf16", 1, 32, 1, 6007, 32, 128, False, offset=6006),
        # an encoder's, odd length, single-precision table, with the gradient that attention hands back for the whole batch
        _bias("bias_train_encoder", True, "fp16", "fp32", 16, 12, 391, 391, 32, 128, True),
        # the largest: the benchmark's sizes with a bias
        _bias("bias_train_long", True, "bf16", "bf16", 8, 16, 2048, 2048, 32, 128, True),
        # a small model's hidden states
        _dropout("dropout_train_tiny", True, "fp16", 256, 512, 0.1, True),
        # rows of a wider tensor, single precision, a width that no vector divides
        _dropout("dropout_train_rows", True, "fp32", 2000, 1003, 0.2, False, pitch=2048),
        # an encoder's hidden states
        _dropout("dropout_train_encoder", True, "fp16", 6256, 768, 0.1, False),
        # a decoder's residual stream
        _dropout("dropout_train_residual", True, "bf16", 16384, 4096, 0.1, True),
    ]


def _log(rng, lo, hi):
    """A whole number from lo..hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _length(rng, lo, hi):
    """A sequence length: odd as often as a multiple of 128."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.6 else max(lo, min(hi, (n + 64) // 128 * 128 or 128))


def draw(rng):
    half = rng.choice(["bf16", "fp16"])
    while True:
        kind = rng.choice(["step", "step", "prompts", "fp32", "train", "train", "bias_step", "bias_train", "bias_train", "dropout", "dropout"])
        sinks = rng.choice([0, 1, 4, 4, 8, 17, 64, 130])
        heads = rng.choice([(8, 8), (16, 4), (32, 8), (32, 4), (12, 12)])
        if kind == "step":
            api, sk = rng.choice(["dense", "padded"]), _length(rng, 50, 16384)
            c = _sink(None, api, False, half, _log(rng, 1, 32), *heads, rng.choice([1, 1, 1, 3]), sk, rng.choice([64, 128, 128, 80]), _log(rng, 16, 4096), sinks,
                      layout=rng.choice(["bhsd", "bshd"]), lo=max(3, sk // 20), hi=sk, lens=rng.randrange(1 << 20))
        elif kind == "prompts":
            c = _sink(None, "compact", False, half, _log(rng, 2, 16), *heads, 0, 0, rng.choice([64, 128, 128, 96]), _log(rng, 32, 1024), sinks,
                      lo=_log(rng, 1, 64), hi=_log(rng, 128, 2048), lens=rng.randrange(1 << 20))
            if sum(_lengths(c)) > 12000:
                continue
        elif kind == "fp32":
            s = _length(rng, 60, 1024)
            c = _sink(None, "dense", True, "fp32", _log(rng, 1, 4), 8, rng.choice([8, 2]), s, s, rng.choice([32, 64, 80, 128]), _log(rng, 16, 512), min(sinks, 8))
        elif kind == "train":
            s = _length(rng, 256, 8192)
            c = _sink(None, "dense", True, half, rng.choice([1, 1, 2]), *heads, s, s, rng.choice([64, 128, 128, 72, 256]), _log(rng, 64, 2048), sinks,
                      layout=rng.choice(["bhsd", "bshd"]))
        elif kind == "bias_step":
            sk = _length(rng, 50, 16384)
            c = _bias(None, False, half, rng.choice([half, "fp32"]), 1, rng.choice([8, 12, 16, 32, 64]), 1, sk, rng.choice([32, 64]), rng.choice([128, 256, 1000]),
                      False, offset=sk - 1)
        elif kind == "bias_train":
            c = _bias(None, True, rng.choice([half, half, "fp32"]), rng.choice(["fp32", "same"]), _log(rng, 1, 16), rng.choice([4, 8, 12, 16]), _length(rng, 30, 2048),
                      _length(rng, 30, 2048), rng.choice([16, 32, 32, 64]), rng.choice([64, 128, 500]), rng.random() < 0.7, offset=rng.choice([0, 0, 0, 5, -3]))
            c["table"] = c["dtype"] if c["table"] == "same" else c["table"]
        else:
            cols = rng.choice([_log(rng, 100, 8192), _log(rng, 16, 1024) * 8])
            c = _dropout(None, True, rng.choice([half, half, "fp32"]), _log(rng, 16, 16384), cols, rng.choice([0.05, 0.1, 0.1, 0.3]), rng.random() < 0.5,
                         pitch=rng.choice([cols, cols, cols + 8, cols + 5]))
        if _plain_elements(c) <= _plain_elements(_LARGEST[c["op"]]):
            return c


def _lengths(c):
    r = random.Random(c["lens"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["b"])]


def _plain_elements(c):
    """What the plain form of a case costs: scores, bias entries or elements."""
    if c["op"] == "sink":
        return c["hq"] * (sum(_lengths(c)) ** 2 if c["api"] == "compact" else c["b"] * c["sq"] * c["sk"]) * (4 if c["train"] else 1) * c["d"]
    return c["b"] * c["h"] * c["sq"] * c["sk"] if c["op"] == "bias" else c["rows"] * c["cols"]


_LARGEST = {c["op"]: c for c in sorted(listed(), key=_plain_elements)}


# ---- inputs ---------------------------------------------------------------------------------------------------
class State:
    pass


def _ends(lengths):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c, s = case, State()
    dt = DTYPES[c["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    s.case = c
    if c["op"] == "sink":
        if c["api"] == "compact":
            lens = _lengths(c)
            s.lens_q = s.lens_k = lens
            # (tokens, heads, head dim) storage, handed over as the (1, heads, tokens, head dim) view
            s.q, s.k, s.v = (rand(1, sum(lens), h, c["d"]).transpose(1, 2) for h in (c["hq"], c["hk"], c["hk"]))
        else:
            s.lens_q = [c["sq"]] * c["b"]
            s.lens_k = _lengths(c) if c["api"] == "padded" else [c["sk"]] * c["b"]
            swap = c["layout"] == "bshd"
            s.q, s.k, s.v, s.dout = (rand(c["b"], *((n, h) if swap else (h, n)), c["d"]).transpose(1, 2) if swap else rand(c["b"], h, n, c["d"])
                                     for h, n in ((c["hq"], c["sq"]), (c["hk"], c["sk"]), (c["hk"], c["sk"]), (c["hq"], c["sq"])))
        if c["api"] != "dense":
            s.ends_q, s.ends_k = _ends(s.lens_q), _ends(s.lens_k)
            s.lens = torch.tensor([s.lens_q, s.lens_k], device="cuda")
        inputs = (s.q, s.k, s.v)
    elif c["op"] == "bias":
        s.table = rand(c["buckets"], c["h"], dtype=DTYPES[c["table"]])
        inputs = (s.table,)
        if c["train"]:
            # what attention hands back: dS, a value times a probability each
            s.dout = rand(c["b"], c["h"], c["sq"], c["sk"]) * (1.0 / c["sk"] ** 0.5)
    else:
        s.x = rand(c["rows"], c["pitch"])[:, :c["cols"]]
        s.residual = rand(c["rows"], c["cols"]) if c["residual"] else None
        s.dout = rand(c["rows"], c["cols"])
        s.seed, s.offset = 1 + seed % 1000003, 1 + seed % 999983
        inputs = (s.x,) + ((s.residual,) if c["residual"] else ())
    s.inputs = inputs
    if c["train"]:
        for t in inputs:
            t.requires_grad_()
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------
def _visible(pos_q, pos_k, c):
    """(queries, keys) truth values from the positions of both in their sequence."""
    p, n = pos_q[..., :, None], pos_k[..., None, :]
    return (n <= p) & ((n > p - c["window"]) | (n < c["sinks"]))


def _mask(s):
    c = s.case
    if c["api"] == "dense":
        pos = torch.arange(c["sk"], device="cuda")
        return _visible(pos[c["sk"] - c["sq"]:], pos, c)
    if c["api"] == "padded":
        n, m = torch.arange(c["sk"], device="cuda"), torch.arange(c["sq"], device="cuda")
        lk = s.lens[1][:, None]
        return (_visible(m + lk - c["sq"], n.expand(c["b"], -1), c) & (n < lk)[:, None, :])[:, None]
    t = torch.arange(s.q.shape[2], device="cuda")
    which = (t[:, None] >= s.ends_q[None, 1:]).sum(1)
    pos = t - s.ends_q[which]
    return _visible(pos, pos, c) & (which[:, None] == which[None, :])


def _plain_sink(s):
    c = s.case
    group, scale = c["hq"] // c["hk"], c["d"] ** -0.5
    q, k, v = (t.detach().float() for t in (s.q, s.k, s.v))
    b, hq, sq, d = q.shape
    q = q.reshape(b, c["hk"], group, sq, d)
    k, v = k[:, :, None], v[:, :, None]
    mask = _mask(s)
    if mask.dim() == 4:
        mask = mask[:, :, None]
    p = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(~mask, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.mul_(torch.where(total > 0, 1 / total, 0.0))
    out = p @ v
    result = out.reshape(b, hq, sq, d).to(s.q.dtype)
    if not c["train"]:
        return result
    do = s.dout.float().reshape(b, c["hk"], group, sq, d)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = (do @ v.transpose(-1, -2)).sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = (ds @ k).reshape(b, hq, sq, d)
    dk = (ds.transpose(-1, -2) @ q).sum(2)
    return result, dq.to(s.q.dtype), dk.to(s.q.dtype), dv.to(s.q.dtype)


def _buckets(c, d):
    """The bucket of each distance d (key's position minus the query's), whole numbers."""
    nb = c["buckets"] // 2 if c["both"] else c["buckets"]
    e = nb // 2
    r = d.abs() if c["both"] else (-d).clamp(min=0)
    # (in 64 bits, with what a logarithm may be off by added: at a border the quotient is a whole number)
    far = e + ((nb - e) * (r.clamp(min=1).double() / e).log() / math.log(c["far"] / e) + 1e-9).floor().long()
    return torch.where(r < e, r, far.clamp(max=nb - 1)) + (nb * (d > 0) if c["both"] else 0)


def _plain_bias(s):
    c = s.case
    h, sq, sk = c["h"], c["sq"], c["sk"]
    m, n = torch.arange(sq, device="cuda"), torch.arange(sk, device="cuda")
    out = s.table.detach().float()[_buckets(c, n[None, :] - m[:, None] - c["offset"])].permute(2, 0, 1).to(DTYPES[c["dtype"]]).expand(c["b"], h, sq, sk)
    if not c["train"]:
        return out
    g = s.dout.float().sum(0)
    # each row with sq zeros in front of it, taken one place further on than the row before: column j is the diagonal n - m = j - sq
    flat = torch.cat([torch.cat([g.new_zeros(h, sq, sq), g], 2).flatten(1), g.new_zeros(h, sq)], 1)
    lines = torch.as_strided(flat, (h, sq, sq + sk), (flat.stride(0), sq + sk + 1, 1))
    sums = lines.sum(1, dtype=torch.float64)
    d = torch.arange(sq + sk, device="cuda") - sq - c["offset"]
    where = (_buckets(c, d)[:, None] == torch.arange(c["buckets"], device="cuda")).double()
    return out, (sums @ where).t().to(s.table.dtype)


def _philox(seed, counter):
    """The four words of each counter, as unsigned 32-bit numbers in 64."""
    low = 0xFFFFFFFF
    c0, c1, c2, c3 = counter & low, (counter >> 32) & low, torch.zeros_like(counter), torch.zeros_like(counter)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c0, c1, c2, c3


def _threshold(p):
    return int(np.trunc((np.float32(p) - np.float32(0.5)) * np.float32(4294967296.0)))


def _plain_dropout(s):
    c = s.case
    n = c["rows"] * c["cols"]
    w = _philox(s.seed, s.offset + torch.arange((n + 3) // 4, device="cuda"))
    word = torch.stack([w[0], w[2], w[1], w[3]], 1).flatten()[:n].view(c["rows"], c["cols"])
    keep = torch.where(word >= 1 << 31, word - (1 << 32), word) > _threshold(c["p"])
    scale = 1.0 / (1.0 - c["p"])
    out = torch.where(keep, s.x.detach().float() * scale, 0.0)
    if c["residual"]:
        out = out + s.residual.detach().float()
    dx = torch.where(keep, s.dout.float() * scale, 0.0).to(s.x.dtype)
    return (out.to(s.x.dtype), dx) + ((s.dout,) if c["residual"] else ())


# ---- one pass -------------------------------------------------------------------------------------------------
def _own_forward(s):
    from aotriton_b200 import autograd

    c = s.case
    if c["op"] == "sink":
        if c["api"] == "dense":
            return autograd.sink_attention(s.q, s.k, s.v, c["window"], c["sinks"])
        return autograd.varlen_sink_attention(s.q, s.k, s.v, s.ends_q, s.ends_k, max(s.lens_q), max(s.lens_k), c["window"], c["sinks"], varlen_type=c["api"])
    if c["op"] == "bias":
        return autograd.relative_position_bias(s.table, c["sq"], c["sk"], batch=c["b"], max_distance=c["far"], bidirectional=c["both"],
                                               query_offset=c["offset"], dtype=DTYPES[c["dtype"]])
    return autograd.dropout(s.x, c["p"], residual=s.residual, philox_seed=s.seed, philox_offset=s.offset)


def _own(s):
    if not s.case["train"]:
        with torch.no_grad():
            return _own_forward(s)
    out = _own_forward(s)
    return (out.detach(),) + torch.autograd.grad(out, s.inputs, s.dout)


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"sink": _plain_sink, "bias": _plain_bias, "dropout": _plain_dropout}[state.case["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------
def _seen(sq, sk, window, sinks):
    """(scores that are not masked, keys that some query sees) of one head."""
    p = np.arange(sk - sq, sk, dtype=np.int64)
    p = p[p >= 0]
    recent = np.maximum(p - window + 1, 0)
    pairs = int((p - recent + 1).sum() + np.minimum(recent, sinks).sum())
    first = int(recent[0]) if len(p) else 0
    return pairs, (sk - first + min(first, sinks)) if len(p) else 0


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "sink":
        ragged = c["api"] != "dense"
        lens_k = _lengths(c) if ragged else [c["sk"]] * c["b"]
        lens_q = lens_k if c["api"] == "compact" else [c["sq"]] * c["b"]
        seen = [_seen(a, b, c["window"], c["sinks"]) for a, b in zip(lens_q, lens_k)]
        pairs, keys = sum(x[0] for x in seen), sum(x[1] for x in seen)
        q, kv = sum(lens_q) * c["hq"] * c["d"], 2 * keys * c["hk"] * c["d"]
        forward = 4 * c["d"] * c["hq"] * pairs
        if not c["train"]:
            return {"bytes": size * (2 * q + kv), "flops": forward}
        # q, k, v and the output's gradient read; the output and the gradients of q, k, v written
        return {"bytes": size * (4 * q + 2 * kv), "flops": 3.5 * forward}
    if c["op"] == "bias":
        entries = c["h"] * c["sq"] * c["sk"]
        table = c["buckets"] * c["h"] * (4 if c["table"] == "fp32" else 2)
        if not c["train"]:
            return {"bytes": size * entries + table, "flops": 0}
        return {"bytes": size * entries * (1 + c["b"]) + 2 * table, "flops": entries * c["b"]}
    n = c["rows"] * c["cols"]
    # x and the residual read, the output written; its gradient read, x's written
    return {"bytes": size * n * (4 + c["residual"]), "flops": 4 * n}


# ---- in 64 bits -----------------------------------------------------------------------------------------------
def _exact_sink(s):
    c = s.case
    scale = 1.0 / math.sqrt(c["d"])
    train = c["train"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in (s.q, s.k, s.v)] if train else []
    at_q = at_k = 0
    for z, (nq, nk) in enumerate(zip(s.lens_q, s.lens_k)):
        packed = c["api"] == "compact"
        bz, iq, ik = (0, slice(at_q, at_q + nq), slice(at_k, at_k + nk)) if packed else (z, slice(0, nq), slice(0, nk))
        at_q, at_k = at_q + nq, at_k + nk
        hidden = torch.ones(nq, nk, dtype=torch.bool, device="cuda")
        here = torch.arange(nk - nq, nk, device="cuda").unsqueeze(1)
        age = here - torch.arange(nk, device="cuda").unsqueeze(0)      # how far behind the query a key lies
        hidden &= ~((age >= 0) & (age < c["window"]))
        hidden[:, :c["sinks"]] &= age[:, :c["sinks"]] < 0
        for h in range(c["hq"]):
            hk = h // (c["hq"] // c["hk"])
            q, k, v = s.q.detach()[bz, h, iq].double(), s.k.detach()[bz, hk, ik].double(), s.v.detach()[bz, hk, ik].double()
            x = (q @ k.T * scale).masked_fill(hidden, -math.inf)
            e = torch.exp(x - x.max(dim=1, keepdim=True).values.clamp(min=-1e300))
            e = e / e.sum(dim=1, keepdim=True).clamp(min=1e-300)
            o = e @ v
            out[bz, h, iq] = o
            if train:
                g = s.dout[bz, h, iq].double()
                grads[2][bz, hk, ik] += e.T @ g
                t = e * (g @ v.T - (g * o).sum(dim=1, keepdim=True)) * scale
                grads[0][bz, h, iq] = t @ k
                grads[1][bz, hk, ik] += t.T @ q
    return (out, *grads) if train else out


def _border(c, k):
    """The smallest distance whose bucket is at least k, from whole numbers alone: r^(nb-e) * e^(k-e) >= e^(nb-e) * far^(k-e)."""
    nb = c["buckets"] // 2 if c["both"] else c["buckets"]
    e = nb // 2
    if k <= e:
        return k
    lo, hi = e, c["far"]
    while lo < hi:
        mid = (lo + hi) // 2
        if mid ** (nb - e) * e ** (k - e) >= e ** (nb - e) * c["far"] ** (k - e):
            hi = mid
        else:
            lo = mid + 1
    return lo


def _exact_bias(s):
    c = s.case
    nb = c["buckets"] // 2 if c["both"] else c["buckets"]
    borders = [_border(c, k) for k in range(1, nb)]
    d = np.arange(c["sk"])[None, :] - np.arange(c["sq"])[:, None] - c["offset"]
    b = np.searchsorted(np.array(borders), np.abs(d) if c["both"] else np.maximum(-d, 0), side="right")
    if c["both"]:
        b = b + nb * (d > 0)
    b = torch.from_numpy(b).cuda()
    t = s.table.detach().double()
    out = t.T[:, b.flatten()].view(1, c["h"], c["sq"], c["sk"]).expand(c["b"], -1, -1, -1)
    if not c["train"]:
        return out
    grad = torch.zeros_like(t)
    for h in range(c["h"]):
        g = s.dout[:, h].double().sum(dim=0)
        for k in range(c["buckets"]):
            grad[k, h] = g[b == k].sum()
    return out, grad


def _exact_dropout(s):
    c = s.case
    n = c["rows"] * c["cols"]
    m = np.uint64(0xFFFFFFFF)
    x = np.uint64(s.offset) + np.arange((n + 3) // 4, dtype=np.uint64)
    w = [x & m, x >> np.uint64(32), np.zeros_like(x), np.zeros_like(x)]
    key = [s.seed & 0xFFFFFFFF, s.seed >> 32]
    for r in range(10):
        lo, hi = w[0] * np.uint64(0xD2511F53), w[2] * np.uint64(0xCD9E8D57)
        w = [(hi >> np.uint64(32)) ^ w[1] ^ np.uint64((key[0] + r * 0x9E3779B9) & 0xFFFFFFFF), hi & m,
             (lo >> np.uint64(32)) ^ w[3] ^ np.uint64((key[1] + r * 0xBB67AE85) & 0xFFFFFFFF), lo & m]
    words = np.empty((len(x), 4), dtype=np.int32)
    for place, i in enumerate((0, 2, 1, 3)):
        words[:, place] = w[i].astype(np.uint32).view(np.int32)
    limit = int((np.float32(c["p"]) - np.float32(0.5)) * np.float32(2.0 ** 32))
    kept = torch.from_numpy(words.reshape(-1)[:n].reshape(c["rows"], c["cols"]) > limit).cuda()
    factor = kept.double() / (1.0 - c["p"])
    out = s.x.detach().double() * factor
    if c["residual"]:
        out += s.residual.detach().double()
    g = s.dout.double()
    return (out, g * factor) + ((g,) if c["residual"] else ())


def exact(case, seed):
    s = prepare(case, seed)
    return {"sink": _exact_sink, "bias": _exact_bias, "dropout": _exact_dropout}[case["op"]](s)
