"""64-bit restatement of what stands around attention in a layer.  TEST INFRASTRUCTURE ONLY.

The visibility of sink attention, the buckets and sums of the learned relative position bias, dropout of hidden states:
dense, from their definitions, with whole-number comparisons where a logarithm would round.
"""
from __future__ import annotations

import numpy as np
import torch

from . import philox


def sink_mask(seqlen_q: int, seqlen_k: int, window: int, sinks: int) -> torch.Tensor:
    """Boolean [Sq, Sk]: query m stands at P = m + Sk - Sq and sees keys n <= P with n > P - window or n < sinks."""
    p = torch.arange(seqlen_q)[:, None] + (seqlen_k - seqlen_q)
    n = torch.arange(seqlen_k)[None, :]
    return (n <= p) & ((n > p - window) | (n < sinks))


def bucket(d: int, buckets: int, max_distance: int, bidirectional: bool) -> int:
    """Bucket of one distance (key minus query): e + floor((nb - e) * log(r / e) / log(max_distance / e)) as the largest k with
    r ** (nb - e) * e ** k >= e ** (nb - e) * max_distance ** k."""
    nb = buckets // 2 if bidirectional else buckets
    r = abs(d) if bidirectional else max(-d, 0)
    second = nb if bidirectional and d > 0 else 0
    e = nb // 2
    if r < e:
        return second + r
    k = 0
    while e + k + 1 < nb and r ** (nb - e) * e ** (k + 1) >= e ** (nb - e) * max_distance ** (k + 1):
        k += 1
    return second + e + k


def bucket_matrix(seqlen_q, seqlen_k, buckets, max_distance, bidirectional, offset) -> torch.Tensor:
    lo = -(seqlen_q - 1) - offset
    line = torch.tensor([bucket(d, buckets, max_distance, bidirectional) for d in range(lo, seqlen_k - offset)])
    m, n = torch.arange(seqlen_q)[:, None], torch.arange(seqlen_k)[None, :]
    return line[n - m - offset - lo]


def relative_bias(table, where) -> torch.Tensor:
    return table.double()[where].permute(2, 0, 1)


def relative_bias_grad(grad, where, buckets) -> torch.Tensor:
    """grad [B, H, Sq, Sk] -> [buckets, H]"""
    g = grad.double().sum(0)
    return torch.stack([torch.where(where == k, g, 0.0).sum((1, 2)) for k in range(buckets)])


def dropout_keep(count: int, dropout_p: float, seed: int, offset: int) -> torch.Tensor:
    with np.errstate(over="ignore"):
        words = philox.philox4x32_10(seed, np.uint64(offset) + np.arange((count + 3) // 4, dtype=np.uint64))
    ordered = words[:, [0, 2, 1, 3]].reshape(-1)[:count]
    keep = np.ones(count, dtype=bool) if dropout_p == 0 else ordered.view(np.int32) > np.int32(philox.dropout_threshold(dropout_p))
    return torch.from_numpy(keep)
