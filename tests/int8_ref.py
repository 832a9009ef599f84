"""The 8-bit projections in 64 bits: codes by exact comparisons, products of
whole numbers, and how far FP32 arithmetic may be from them."""

import numpy as np

EPS32 = 2.0 ** -24                                   # half a step of FP32, relative
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}


def codes(t):
    """Codes [rows, Kp] and scales (FP32) of rows of FP32 values."""
    t = np.asarray(t, np.float32)
    top = np.abs(t).max(1, initial=0.0) if t.shape[1] else np.zeros(len(t), np.float32)
    bad = ~np.isfinite(t).all(1)
    x = np.where(bad[:, None], 0, t).astype(np.longdouble)
    m = np.where(bad, 0, top).astype(np.longdouble)
    safe = np.where(m > 0, m, 1)[:, None]
    lo = np.floor(127 * x / safe)                    # 64 bits of mantissa: floor is right or one off at a whole number
    lo = np.where((lo + 1) * safe <= 127 * x, lo + 1, lo)
    lo = np.where(lo * safe > 127 * x, lo - 1, lo)
    twice = 254 * x - (2 * lo + 1) * safe            # sign of 127 x / top - (lo + 1/2), exact
    q = np.where((twice > 0) | ((twice == 0) & (lo % 2 != 0)), lo + 1, lo)
    q = np.where(m[:, None] > 0, q, 0).astype(np.int8)
    kp = -(-t.shape[1] // 128) * 128
    out = np.zeros((len(t), kp), np.int8)
    out[:, : t.shape[1]] = q
    with np.errstate(all="ignore"):
        scale = np.where(bad, np.float32(np.nan), top / np.float32(127)).astype(np.float32)
    return out, scale


def linear(x, w, ws, gain=None, eps=None, bias=None, residual=None, swiglu=False, bf16=False):
    """(out, bound): the projection in 64 bits from FP32 values x and codes w, and how far FP32
    arithmetic may be from it before the output's own rounding.

    Every FP32 operation is off by at most half a step, EPS32 of its result.  The sum of squares adds
    at most K/512 + 14 positive terms one on another (8 in a lane, 6 exchanges, the blocks), so it is
    within (K/512 + 14) EPS32; root and quotient halve that and add two steps, the mean and eps two more
    halves; top / 127, the product with it, the whole sum as FP32 and two products by scales: five
    more.  silu(g) = g / (1 + e^-g): the GPU's power of two and its reciprocal are each within a step (2 EPS32) of the
    result; the power's correction adds 2, the sum, the product and the last product 1 each: 9.  For BF16 outputs the
    exponent -g log2(e) is rounded (EPS32 of it, and 0.22 for the constant: together 1.25 |g| ln 2 log2(e) EPS32 of
    the power).  An error r of g moves silu by at most (1 + |g|) r."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        t = x if gain is None else (x * np.asarray(gain, np.float32)).astype(np.float32)
    q, s = codes(t)
    k = x.shape[1]
    s = s.astype(np.float64)
    rel = 5.0
    if eps is not None:
        s = s / np.sqrt((x.astype(np.float64) ** 2).sum(1) / k + np.float64(np.float32(eps)))
        rel += (k / 512 + 14) / 2 + 3
    rel *= EPS32
    acc = q.astype(np.float64) @ w.astype(np.float64).T   # below 2^53: exact
    y = acc * s[:, None] * ws.astype(np.float64)
    off = np.abs(y) * rel
    if bias is not None:
        y = y + bias.astype(np.float64)
        off = off + np.abs(y) * EPS32
    if swiglu:
        n = y.shape[1] // 2
        g, u, og, ou = y[:, :n], y[:, n:], off[:, :n], off[:, n:]
        with np.errstate(over="ignore"):
            a = g / (1 + np.exp(-g))
        # |d silu| <= 1.1, and where silu is tiny its slope is at most (1 + |g|) of its value over |g|
        slope = np.minimum(1.1, np.abs(a) * (1 + np.abs(g)) / np.maximum(np.abs(g), 1e-300))
        slope = np.where(np.abs(g) < 1, 1.1, slope)
        oa = slope * og * 1.01 + np.abs(a) * (9 + (1.25 * np.abs(g) if bf16 else 0)) * EPS32
        y = a * u
        off = oa * np.abs(u) + np.abs(a) * ou + oa * ou + np.abs(y) * EPS32
    if residual is not None:
        y = y + residual.astype(np.float64)
        off = off + np.abs(y) * EPS32
    # where scales are denormal each of the products loses up to 2^-149 of its own
    return y, off * 1.01 + 2.0 ** -148 * (1 + np.abs(ws.astype(np.float64)).max(initial=0.0))
