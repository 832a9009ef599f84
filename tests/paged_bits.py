"""Inputs of the paged operators on which low bits decide: what the kernels' cutting of FP32 values into
BF16 parts may leave out, and bounds narrow enough to see a part that is missing.

The kernels' arithmetic, in 64 bits but with the parts cut as they cut them, is here too: a
part dropped in it has to fail the bound."""

import math

import numpy as np
import torch

import paged_ref as ref
from paged_ref import HALF_STEP, Setup

EPS = 2.0 ** -24


def cut(x, n):
    """x as n BF16 parts that add up to it: cut to 8 bits, the rest cut again; the second of two rounds
    to nearest, as does the only one."""
    rest, out = np.asarray(x, np.float32), []
    for i in range(n):
        if i == n - 1 and n < 3:
            part = torch.from_numpy(np.ascontiguousarray(rest)).to(torch.bfloat16).float().numpy()
        else:
            part = (rest.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        out.append(part.astype(np.float64))
        rest = rest - part
    return out


def near_ties(seqs, heads, hd, xd, kd, width=None, seed=0, level=0):
    """Scores that FP32 and BF16 products give exactly, close to each other (and to level^2 / 16), and values of -1 and
    1: a row's result is a difference of weights.  Returns the inputs and the scale."""
    u = Setup(seqs, *heads, hd, 16, xd, kd, width=width, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)

    def pick(like, values):
        return torch.tensor(values)[torch.randint(len(values), like.shape, generator=g)].to(like.dtype)

    u.q, u.k = pick(u.q, [-0.5, 0.0, 0.5]), pick(u.k, [-1.0, -0.5, 0.0, 0.5, 1.0])
    u.v = pick(u.v, [-1.0, 1.0])
    if level:
        u.q[..., -1], u.k[..., -1] = level, level
    return u, 2.0 ** -4


def low_queries(seqs, heads, hd, width=None, seed=0):
    """FP32 queries in pairs of dims (x, x without its last 8 bits) against keys (c, -c) of a BF16 cache: a score is
    what the last 8 bits give, and exact where the products of each part add up by themselves (over an
    FP32 cache whole products do: four x reach 8, whose step is 2^-20, and the last 8 bits are rounded away).
    Returns the inputs and the scale that makes it count."""
    u = Setup(seqs, *heads, hd, 16, torch.float32, torch.bfloat16, width=width, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    x = torch.rand(*u.q.shape[:-1], hd // 2, generator=g) + 1.0
    hi = (x.view(torch.int32) & ~0xFF).view(torch.float32)
    c = torch.tensor([-1.0, -0.5, 0.5, 1.0])[torch.randint(4, (*u.k.shape[:-1], hd // 2), generator=g)]
    u.q = torch.stack((x, hi), -1).flatten(-2)
    u.k = torch.stack((c, -c), -1).flatten(-2).to(torch.bfloat16)
    u.v = torch.where(torch.rand(u.v.shape, generator=g) < 0.5, -1.0, 1.0).to(torch.bfloat16)
    return u, 2.0 ** 14 / math.sqrt(hd)


def low_products(seqs, heads, hd, swap=False, seed=0):
    """FP32 queries and keys whose scores are made of the products of one side's second part and the other's third.

    Groups of four of the first 16 dims hold (256 + a, -256, -a, 0) . (k, k, 65792, 0) = a b with k = 65792 + b and a, b
    0 or 1: the parts of k are 65536, 256 and b, those of 256 + a are 256 and a.  All other products of parts cancel as
    they are added up (part by part, whole numbers up to 2^26), so a score is the number of groups with a = b = 1, exactly.
    swap: keys and queries change places.  Returns the inputs and the scale."""
    u = Setup(seqs, *heads, hd, 16, torch.float32, torch.float32, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)

    def bit(like):
        return torch.randint(2, (*like.shape[:-1], 4), generator=g).float()

    two, three = (u.k, u.q) if swap else (u.q, u.k)
    a, k = bit(two), 65792.0 + bit(three)
    two.zero_()[..., :16] = torch.stack((256.0 + a, torch.full_like(a, -256.0), -a, 0.0 * a), -1).flatten(-2)
    three.zero_()[..., :16] = torch.stack((k, k, torch.full_like(k, 65792.0), 0.0 * k), -1).flatten(-2)
    u.mass.zero_()
    return u, 0.5


def simulate(u, scale, window, q_parts, p_parts):
    """out of the kernels' arithmetic with q and the weights in so many parts, the rest in 64 bits."""
    out = np.full((u.T, u.Hq, u.hd), np.nan)
    q = sum(cut(u.q.float().numpy(), q_parts)[::-1])
    for s in range(u.S):
        n = int(u.lens[s])
        for h in range(u.Hkv):
            k, v = u.keys(u.k, s, h, n), u.keys(u.v, s, h, n)
            for m in u.rows(s):
                see = ref.seen(u.slot(s, m), window, 0)
                for a in range(h * u.G, (h + 1) * u.G):
                    x = scale * (k[see] @ q[m, a])
                    p = np.exp(x - x.max()).astype(np.float32)
                    out[m, a] = sum(cut(p, p_parts)) @ v[see] / p.sum(dtype=np.float64)
    return torch.from_numpy(out).to(u.xd).double().numpy()


def out_bound(u, scale, window):
    """(exact out, how far an output may be) with scores that are exact.  A weight: the factor log2 e and
    its product off by a step of the exponent, the difference from the maximum by as much, and that of an
    earlier maximum (5 S steps of 2^-24, S the largest difference of two scores of a row: weights and sums refer to one and the
    same rounded maximum, so its own size does not count), the exponential and up to one change of
    the maximum (8).  Those count once in the sum over values, once in the sum of weights; n additions
    and the factors in common follow (8).  BF16 activations: weights of 16 bits, 2^-16 of each, and the output's rounding."""
    want, _, weight, size = ref.attention(u, scale, window, 0)
    _, S, n = scores_of(u, scale, window)
    fine = (2.0 * (5.0 * S + 8.0) + n + 8.0) * EPS * weight
    if u.xd == torch.bfloat16:
        fine = fine + 2.0 ** -16 * weight
        fine = fine + HALF_STEP[u.xd] * (np.abs(want) + fine)
    return want, fine + EPS * np.abs(want)


def scores_of(u, scale, window):
    """The largest |score| that a row sees, the largest difference of two of a row, and the most keys that one sees."""
    top, apart, most, q = 0.0, 0.0, 0, u.q.double().numpy()
    for s in range(u.S):
        for h in range(u.Hkv):
            k = u.keys(u.k, s, h, int(u.lens[s]))
            for m in u.rows(s):
                see = ref.seen(u.slot(s, m), window, 0)
                if not see:
                    continue
                x = scale * (k[see] @ q[m, h * u.G: (h + 1) * u.G].T)
                top, apart, most = max(top, float(np.abs(x).max())), max(apart, float(np.ptp(x, 0).max())), max(most, len(see))
    return top, apart, most


def simulate_mass(u, scale, lse, keep):
    """The accounts with the products of parts (i of q, j of k) for which keep(i, j)."""
    out = np.zeros(u.mass.shape)
    qs = cut(u.q.numpy(), 3)
    for s in range(u.S):
        n = int(u.lens[s])
        e, j = u.table[s, np.arange(n) // u.page], np.arange(n) % u.page
        for h in range(u.Hkv):
            ks = [p[e, h, j] for p in cut(u.k.float().numpy(), 3)]
            for m in u.rows(s):
                see = u.slot(s, m) + 1
                for a in range(h * u.G, (h + 1) * u.G):
                    x = sum(ks[b][:see] @ qs[i][m, a] for i in range(3) for b in range(3) if keep(i, b))
                    np.add.at(out, (e[:see], h, j[:see]), np.exp(scale * x - lse[m, a]))
    return out


def mass_bound(u, scale, lse):
    """(exact accounts, how far one may be) with scores that are exact.  A weight: the score's scaling, the
    difference from lse and the factor log2 e off by a step of the exponent each (3 A), the exponential (2); then one
    addition per term."""
    want, terms = ref.mass(u, lse, scale)
    A = scores_of(u, scale, 0)[0] + float(np.abs(lse).max())
    return want, (3.0 * A + 2.0 + terms) * EPS * want
