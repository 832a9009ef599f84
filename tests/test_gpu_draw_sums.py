"""Sums of the sampler by row where they are hardest: tails of many light values below one that has nearly all the weight,
rows whose parts lie far below each other, and draws from the far end of the kept sum.  A row has the same bits however many rows
share its call."""

import numpy as np
import pytest
import torch

import draw_ref as ref
from test_gpu_draw import words_of

pytestmark = pytest.mark.gpu

BITS = lambda v: min(46, 62 - int(np.ceil(np.log2(v))))  # noqa: E731


@pytest.fixture(scope="module")
def ops(hip_device):
    from soraku_amd import ops as O

    return O


def draw(ops, dev, x, u, allowed=None, **p):
    rows = x.shape[0]
    logprob, kept = torch.full((rows,), 7.0, device=dev), torch.full((rows,), -5, device=dev, dtype=torch.int32)
    out = torch.full((rows,), -77, device=dev, dtype=torch.int64)
    ops.sample_rows(x.shape[1])(x, torch.as_tensor(u, dtype=torch.float64).to(dev), out=out, logprob=logprob, kept=kept,
                                allowed=allowed, **{k: t.to(dev) for k, t in p.items()})
    return out.cpu().numpy(), logprob.cpu().numpy(), kept.cpu().numpy()


def slack(v, c):
    """Ids that a draw from a tail of equal values e^c may be off by.  The tail lies in one bucket and the largest in another,
    each sum rounded to the nearest unit, the draw's part of the whole rounded down to one: 2 units of 2^-bits of a power of two that is
    at most twice the largest (1); then a weight's own rounding, 2^-bits of it, over at most v of them."""
    return 2 * 2.0 ** (1 - BITS(v)) / np.exp(c) + v * 2.0 ** -BITS(v) + 1


TAILS = [(40000, -32.1), (40000, -31.0), (151936, -30.6), (1 << 20, -29.3), (1 << 20, -36.0), (16000, -33.0), (9000, -20.0)]


@pytest.mark.parametrize("rows", [1, 16, 130])
@pytest.mark.parametrize("blocked", ["none", "bits", "infinite"])
@pytest.mark.parametrize("v,c", TAILS)
def test_one_peak_and_a_flat_tail(ops, hip_device, v, c, blocked, rows):
    c = float(np.float32(c))
    rng = np.random.default_rng(v)
    us = [1 - 2.0 ** -53, 1.0, 2.0, 1 - 2.0 ** -24, 0.5, 1 - 2.0 ** -40, 1 - 2.0 ** -30]
    u = np.array([us[i % len(us)] for i in range(rows)]) if rows > 1 else None
    peak = 17
    on = np.ones(v, bool)
    if blocked != "none":
        on = rng.random(v) < 0.7
        on[peak], on[v - 1] = True, False
    x = torch.full((rows, v), c)
    x[:, peak] = 0.0
    if blocked == "infinite":
        x[:, torch.from_numpy(~on)] = torch.tensor([-float("inf"), float("nan")])[torch.arange(int((~on).sum())) % 2]
    x = x.to(hip_device)
    bits = words_of(on[None]).to(hip_device) if blocked == "bits" else None
    tail = np.nonzero(on)[0]
    tail = tail[tail != peak]
    w = np.exp(c)
    total = 1 + len(tail) * w
    for one in us if rows == 1 else [None]:
        uu = np.array([one]) if rows == 1 else u
        tok, lp, kept = draw(ops, hip_device, x, uu, bits)
        for r in range(rows):
            assert kept[r] == len(tail) + 1
            T = min(uu[r], 1.0) * total
            at = min(int((T - 1) / w), len(tail) - 1) if T >= 1 else -1
            assert 0 <= tok[r] < v and on[tok[r]], (r, uu[r], tok[r])
            got = -1 if tok[r] == peak else int(np.searchsorted(tail, tok[r]))
            assert abs(got - at) <= slack(v, c), (r, uu[r], got, at)
            want = (0.0 if got < 0 else c) - np.log1p(len(tail) * w)
            # the sum within 2 units, then one rounding
            assert abs(lp[r] - want) <= abs(want) * 2.0 ** -24 + 2.0 ** (3 - BITS(v)), (r, lp[r], want)


@pytest.mark.parametrize("v,c", TAILS)
def test_filters_among_a_flat_tail(ops, hip_device, v, c):
    """top-p and min-p whose bounds lie in the tail, or either side of it."""
    c = float(np.float32(c))
    x = torch.full((6, v), c)
    x[:, v // 2] = 0.0
    n, w = v - 1, np.exp(c)
    p = dict(top_p=torch.tensor([1 - 2.0 ** -24, 1 - 2.0 ** -23, 0, 0, 1 - 2.0 ** -24, 0.5], dtype=torch.float32),
             min_p=torch.tensor([0, 0, 0.5 * w, 2 * w, 0.5 * w, 0.5 * w], dtype=torch.float32))
    tok, _, kept = draw(ops, hip_device, x.to(hip_device), [1.0] * 6, **p)
    total = 1 + n * w
    for r in range(6):
        tp, mp = float(p["top_p"][r]), float(p["min_p"][r])
        want = n + 1
        if tp:
            T = tp * total
            want = 1 if T < 1 else min(int((T - 1) / w) + 2, n + 1)
        exact = not tp or tp == 0.5 or T < 1 - 1e-9
        if mp > w:
            want, exact = 1, True
        assert kept[r] == want if exact else abs(kept[r] - want) <= slack(v, c), (r, kept[r], want)
        at = 0 if tok[r] == v // 2 else 1 + tok[r] - (tok[r] > v // 2)   # place in the order of values
        assert 0 <= at < kept[r] and kept[r] - 1 - at <= slack(v, c), (r, tok[r], kept[r])


@pytest.mark.parametrize("v", [20000, 40000, 151936])
def test_the_end_of_the_draw_is_kept(ops, hip_device, v):
    """top-k ends among many equal light values, min-p a little further down: a draw from the end of the sum
    stays within what top-k keeps."""
    rows, k = 16, 1500
    rng = np.random.default_rng(v)
    x = np.full((rows, v), -45.0, np.float32)
    p = dict(top_k=torch.full((rows,), k, dtype=torch.int32), min_p=torch.full((rows,), float(np.exp(-28.0))))
    for r in range(rows):
        ids = v // 5 + rng.permutation(v - v // 5)[: k - 1 + 100]
        x[r, 0] = 0.0
        x[r, ids[: k - 1]] = -25.0 - 0.01 * r
        x[r, ids[k - 1:]] = -28.0
    for u in (1 - 2.0 ** -53, 1.0, 3.0):
        tok, _, kept = draw(ops, hip_device, torch.from_numpy(x).to(hip_device), [u] * rows, **p)
        assert (kept == k).all()
        # the end of the sum is among the light ones, whose part of it is some 2e-8
        assert ((x[np.arange(rows), tok] > -27.0) & (tok != 0)).all(), x[np.arange(rows), tok]


@pytest.mark.parametrize("v", [17000, 40000, 151936])
def test_a_row_has_the_same_bits_in_any_call(ops, hip_device, v):
    """Rows cut in ten, some, two parts and whole."""
    rng = np.random.default_rng(v)
    rows = 200
    x = rng.standard_normal((rows, v)).astype(np.float32) * rng.choice([1.0, 2.5, 9.0], (rows, 1)).astype(np.float32)
    x[1::3] -= np.linspace(0, 40, v).astype(np.float32)
    x[2::9, 5] += 30.0
    x[3::9] = np.round(x[3::9])                      # many equal ones
    x = torch.from_numpy(x).to(hip_device)
    p = dict(temperature=rng.choice([0.6, 1.0, 1.4], rows), top_p=rng.choice([0.0, 0.9, 0.999999], rows),
             min_p=rng.choice([0.0, 1e-12, 1e-5], rows))
    p = {n: torch.from_numpy(t.astype(np.float32)) for n, t in p.items()}
    p["top_k"] = torch.from_numpy(rng.choice([0, 50, 1024, 1025, 9000, v - 3], rows).astype(np.int32))
    u = rng.random(rows)
    u[:6] = [1 - 2.0 ** -53, 1.0, 0.0, 1 - 2.0 ** -30, 0.9999, 2.0]
    whole = draw(ops, hip_device, x, u, **p)
    for n in (1, 3, 25, 70, 120):
        for at in (0, 7, rows - n):
            s = slice(at, at + n)
            part = draw(ops, hip_device, x[s], u[s], **{k: t[s] for k, t in p.items()})
            assert (part[0] == whole[0][s]).all() and (part[2] == whole[2][s]).all()
            assert (part[1].view(np.int32) == whole[1][s].view(np.int32)).all()


@pytest.mark.parametrize("v", [40, 3000, 20000])
def test_logarithms_are_not_above_0(ops, hip_device, v):
    """Of several kept ones whose others weigh next to nothing."""
    rng = np.random.default_rng(v)
    rows = 100
    x = np.full((rows, v), -90.0, np.float32)
    x[np.arange(rows), rng.integers(0, v, rows)] = rng.standard_normal(rows)
    t = rng.uniform(0.5, 1.5, rows).astype(np.float32)
    tok, lp, kept = draw(ops, hip_device, torch.from_numpy(x).to(hip_device), rng.random(rows), temperature=torch.from_numpy(t))
    assert (tok == x.argmax(1)).all() and (kept == v).all()
    assert (lp <= 0).all() and (lp > -1e-9).all(), lp.max()


@pytest.mark.parametrize("v", [300, 5000, 40000])
def test_close_values_and_light_ones(ops, hip_device, v):
    """Bounds among thousands of close values, with light ones below them, against the row sorted in 64 bits."""
    rng = np.random.default_rng(v + 9)
    rows = 24
    x = (-3.0 + rng.integers(0, 3000, (rows, v)) * 2.0 ** -22).astype(np.float32)
    x[:, v // 3: v // 2] -= 14.0
    p = dict(top_k=torch.from_numpy(rng.choice([0, 40, 1000, v // 2, v - 5], rows).astype(np.int32)),
             top_p=torch.from_numpy(rng.choice([0.0, 0.3, 0.97, 0.99999], rows).astype(np.float32)),
             min_p=torch.from_numpy(rng.choice([0.0, 0.9997, 1e-7, 1e-6], rows).astype(np.float32)))
    u = rng.random(rows)
    tok, lp, kept = draw(ops, hip_device, torch.from_numpy(x).to(hip_device), u, **p)
    known = 0
    for r in range(rows):
        t, l, n, margin, sure = ref.row(x[r], u[r], **{k: a[r].item() for k, a in p.items()})
        if sure:
            assert kept[r] == n
        if sure and margin > ref.safe(v):
            known += 1
            assert tok[r] == t and abs(lp[r] - l) <= abs(l) * 2.0 ** -24 + 1e-8
    assert known >= rows * 3 // 4
