"""The paged-cache operators in 64 bits on the CPU, one sequence, head and row at
a time, and random inputs for them."""

import math

import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}   # of a rounding, relative

# (new tokens, length) of the sequences, heads of 64 with a key head each and width of the table at pages of 16, and the attention kernel
# that takes them by type: with many heads a few short sequences reach the kernels of many rows
MANY_HEADS = [
    ([(150, 150), (40, 200), (9, 90)], 64, 13, {"f32": ("rows", 2), "f32_on_bf16": ("tiles", 0), "bf16": ("tiles", 0)}),
    ([(20, 90), (17, 300), (31, 31), (2, 40)], 64, 19, {"f32": ("rows", 1), "f32_on_bf16": ("few", 2), "bf16": ("few", 2)}),
]


class Setup:
    """Random pools, a table of pages in random order and packed new tokens.
    ``seqs``: (new tokens, length with them) of each sequence; ``pad``: rows behind the last."""

    def __init__(self, seqs, Hq=4, Hkv=2, hd=16, page=16, xd=torch.float32, kd=torch.float32, width=None, pad=0, spare=3,
                 seed=0, spread=1.4):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.seqs, self.Hq, self.Hkv, self.hd, self.page, self.xd, self.kd = seqs, Hq, Hkv, hd, page, xd, kd
        self.S, self.G = len(seqs), Hq // Hkv
        self.starts = np.concatenate(([0], np.cumsum([n for n, _ in seqs]))).astype(np.int32)
        self.lens = np.array([n for _, n in seqs], np.int32)
        self.T = int(self.starts[-1]) + pad
        self.width = width or max(1, -(-max(n for _, n in seqs) // page))
        self.n_pages = self.S * self.width + spare
        self.table = rng.permutation(self.n_pages)[: self.S * self.width].reshape(self.S, self.width).astype(np.int32)
        self.free = np.setdiff1d(np.arange(self.n_pages), self.table).astype(np.int32)

        def rand(*shape, dtype, scale):
            return (torch.randn(*shape, generator=g) * scale).to(dtype)

        self.k = rand(self.n_pages, Hkv, page, hd, dtype=kd, scale=spread)
        self.v = rand(self.n_pages, Hkv, page, hd, dtype=kd, scale=1.0)
        self.q = rand(self.T, Hq, hd, dtype=xd, scale=spread)
        self.qkv = rand(self.T, (Hq + 2 * Hkv) * hd, dtype=xd, scale=0.7)
        self.mass = rand(self.n_pages, Hkv, page, dtype=torch.float32, scale=1.0).abs()
        self.rng = rng

    def rows(self, s):
        return range(int(self.starts[s]), int(self.starts[s + 1]))

    def slot(self, s, m):
        return int(self.lens[s]) - self.seqs[s][0] + m - int(self.starts[s])

    def keys(self, pool, s, h, n):
        """Slots 0 .. n of one head in 64 bits (NaN where the page is none)."""
        j = np.arange(n)
        e = self.table[s, j // self.page]
        ok = (e >= 0) & (e < self.n_pages)
        out = pool[torch.from_numpy(np.where(ok, e, 0)).long(), h, torch.from_numpy(j % self.page)].double().numpy()
        out[~ok] = np.nan
        return out

    def on(self, dev):
        """Device copies, by name."""
        d = {k: getattr(self, k).to(dev) for k in ("k", "v", "q", "qkv", "mass")}
        for k in ("starts", "lens", "table"):
            d[k] = torch.from_numpy(np.ascontiguousarray(getattr(self, k))).to(dev)
        return d


def seen(p, window, sinks):
    """The slots that the token at slot p sees."""
    return [j for j in range(p + 1) if not window or j > p - window or j < sinks]


def attention(u, scale=None, window=0, sinks=0):
    """out, lse, and sum p |v| and the largest scale sum |q k| of every row (what errors are relative to)."""
    scale = u.hd ** -0.5 if scale is None else scale
    out = np.full((u.T, u.Hq, u.hd), np.nan)
    lse, weight, size = np.full((u.T, u.Hq), np.nan), np.zeros((u.T, u.Hq, u.hd)), np.zeros((u.T, u.Hq))
    q = u.q.double().numpy()
    for s in range(u.S):
        n = int(u.lens[s])
        for h in range(u.Hkv):
            k, v = u.keys(u.k, s, h, n), u.keys(u.v, s, h, n)
            for m in u.rows(s):
                see = seen(u.slot(s, m), window, sinks)
                for a in range(h * u.G, (h + 1) * u.G):
                    if not see:
                        out[m, a], lse[m, a] = 0.0, -math.inf
                        continue
                    with np.errstate(all="ignore"):
                        x = scale * (k[see] @ q[m, a])
                        top = x.max()
                        p = np.exp(x - top)
                        lse[m, a] = top + math.log(p.sum()) if np.isfinite(p.sum()) else np.nan
                        p /= p.sum()
                        out[m, a], weight[m, a] = p @ v[see], p @ np.abs(v[see])
                        size[m, a] = scale * (np.abs(k[see]) @ np.abs(q[m, a])).max()
    return out, lse, weight, size


def mass(u, lse, scale=None, window=0, sinks=0):
    """The accounts after a call, and the terms added to each."""
    scale = u.hd ** -0.5 if scale is None else scale
    out, terms = u.mass.double().numpy().copy(), np.zeros(u.mass.shape)
    q, lse = u.q.double().numpy(), np.asarray(lse, np.float64)
    for s in range(u.S):
        n = int(u.lens[s])
        for h in range(u.Hkv):
            k = u.keys(u.k, s, h, n)
            for m in u.rows(s):
                see = np.array(seen(u.slot(s, m), window, sinks), int)
                for a in range(h * u.G, (h + 1) * u.G) if len(see) else ():
                    w = np.exp(scale * (k[see] @ q[m, a]) - lse[m, a])
                    e = u.table[s, see // u.page]
                    ok = (e >= 0) & (e < u.n_pages)
                    np.add.at(out, (e[ok], h, see[ok] % u.page), w[ok])
                    np.add.at(terms, (e[ok], h, see[ok] % u.page), 1)
    return out, terms


def append(u, q_gain, k_gain, inv_freq, positions, eps):
    """q, K, V and the accounts after a call, all in 64 bits."""
    x = u.qkv.double().numpy().reshape(u.T, u.Hq + 2 * u.Hkv, u.hd)
    k, v, mass = u.k.double().numpy().copy(), u.v.double().numpy().copy(), u.mass.double().numpy().copy()
    q = np.full((u.T, u.Hq, u.hd), np.nan)
    half = u.hd // 2
    for s in range(u.S):
        for m in u.rows(s):
            y = x[m].copy()
            ang = float(positions[m]) * inv_freq.astype(np.float64)
            for h in range(u.Hq + u.Hkv):
                if q_gain is not None:
                    y[h] = y[h] / math.sqrt((y[h] ** 2).mean() + eps) * (q_gain if h < u.Hq else k_gain)
                a, b = y[h, :half].copy(), y[h, half:].copy()
                y[h, :half], y[h, half:] = a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)
            q[m] = y[: u.Hq]
            j = u.slot(s, m)
            e = int(u.table[s, j // u.page]) if 0 <= j < u.width * u.page else -1
            if 0 <= e < u.n_pages:
                k[e, :, j % u.page], v[e, :, j % u.page] = y[u.Hq: u.Hq + u.Hkv], y[u.Hq + u.Hkv:]
                mass[e, :, j % u.page] = 0.0
    return q, k, v, mass


def evict(u, keep, sinks, recent):
    """(new lens, kept slots)."""
    kept = np.full((u.S, u.Hkv, keep), -1, np.int32)
    for s in range(u.S):
        n = int(u.lens[s])
        for h in range(u.Hkv):
            w = u.keys(u.mass, s, h, n)
            order = sorted(range(n), key=lambda j: (not (j < sinks or j >= n - recent), not np.isnan(w[j]), -w[j], j))
            best = sorted(order[: min(n, keep)])
            kept[s, h, : len(best)] = best
    return np.minimum(u.lens, keep), kept


def attention_bound(u, out, weight, size, n_keys, rounds_p):
    """How far an output may be: a score's sum of hd products and its few more roundings shift every
    weight by at most twice that, the sums over keys round once per key, weights may be
    rounded to the cache's type once (``rounds_p``), and the output is rounded at the end."""
    half = 2.0 ** -24
    shift = 2.0 * (u.hd + 8) * half * (1.0 + size)[..., None]
    rel = 2.0 * shift + (n_keys + 16) * half + (2.0 * HALF_STEP[torch.bfloat16] if rounds_p else 0.0)
    return rel * weight + HALF_STEP[u.xd] * np.abs(out) + 1e-30
