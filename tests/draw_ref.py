"""Sampling by row in 64 bits: the whole row sorted, weights summed in order.

``margin`` says how near a row's bounds come to a sum or weight of one of its values, as a part of the whole sum: a
draw is determined where it is above what rounding can move sums by (``safe``)."""

import numpy as np


def safe(v):
    """Weights are rounded to whole multiples of 2^-bits of a power of two that is at most twice the largest weight, bits =
    min(46, 62 - log2 v): each is off by at most half of one, at random; 16 sqrt(v) of them is 55 standard deviations of
    their sum (0.29 sqrt(v)), and the whole is at least the largest weight.  The reference's own sums in 64 bits are off by
    less (at most v 2^-53, as they fall sqrt(v) 2^-53).  Past 16,384 values up to 10 workgroups each leave 1,504 sums cut to
    whole multiples, less than one each."""
    cut = 10 * 1504 if v > 16384 else 0
    return 2 * (16 * v ** 0.5 + cut) * 2.0 ** -min(46, 62 - int(np.ceil(np.log2(max(v, 2)))))


def merge(logits, scale):
    """FP32 uncond + scale (cond - uncond) of [rows, 2, V], each operation rounded."""
    c, u = np.asarray(logits[:, 0], np.float32), np.asarray(logits[:, 1], np.float32)
    s = np.asarray(scale, np.float32)[:, None]
    with np.errstate(all="ignore"):
        return (u + (s * (c - u)).astype(np.float32)).astype(np.float32)


def row(x, u, temperature=1.0, top_k=0, top_p=0.0, min_p=0.0, allowed=None):
    """(token, logprob, kept, margin, sure) of one row of FP32 values; sure: whether `kept` is determined."""
    x = np.asarray(x, np.float32)
    ok = np.isfinite(x)
    if allowed is not None:
        ok &= allowed
    ids = np.nonzero(ok)[0]
    if not len(ids):
        return -1, -np.inf, 0, np.inf, True
    t = np.float32(temperature)
    if not t > 0:
        return int(ids[np.argmax(x[ids])]), 0.0, 1, np.inf, True
    big = np.finfo(np.float32).max
    with np.errstate(all="ignore"):
        y = np.clip((x[ids] / t).astype(np.float32), -big, big).astype(np.float64)
    order = np.lexsort((ids, -y))
    ids, y = ids[order], y[order]
    n, SAFE = len(y), safe(len(x))
    with np.errstate(all="ignore"):
        w = np.exp(y - y[0])
    keep, margin, sure = n, np.inf, True
    if 0 < top_k < n:
        keep = int((y >= y[top_k - 1]).sum())
    W = np.cumsum(w[:keep])
    n_k = keep
    p = float(np.float32(top_p))
    if 0 < p < 1:
        T = p * W[-1]
        n_p = min(int(np.searchsorted(W, T, side="right")) + 1, n_k)
        sure &= bool(np.abs(W - T).min() / W[-1] > SAFE)
        keep = min(keep, n_p)
    m = float(np.float32(min_p))
    if 0 < m <= 1:
        keep = min(keep, int((w >= m).sum()))
        off = np.abs(w[:n_k] / m - 1)
        sure &= bool((off[off > 0].min(initial=1) > 1e-9))
    total = W[keep - 1]
    T = min(max(float(u), 0.0), 1.0) * total
    j = min(int(np.searchsorted(W[:keep], T, side="right")), keep - 1)
    if T > 0:                                        # at 0 the first one is the first whose sum passes
        margin = np.abs(W[:keep] - T).min() / total
        if T >= total:
            margin = np.inf if w[keep - 1] / total > SAFE else 0.0
    return int(ids[j]), float(y[j] - y[0] - np.log(total)), keep, float(margin), sure
