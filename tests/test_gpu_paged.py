"""Attention over a cache in pages on the GPU, each operator against its formula
in 64 bits (paged_ref.py): types, head layouts, pages, lengths from none on,
windows that leave little, rows behind the last sequence, and what lies where
nobody may look."""

import numpy as np
import pytest
import torch

import paged_ref as ref
from paged_ref import HALF_STEP, Setup

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TYPES = {"f32": (F32, F32), "f32_on_bf16": (F32, BF16), "bf16": (BF16, BF16)}


@pytest.fixture(scope="module")
def ops(hip_device):
    from soraku_amd import ops as O

    return O


def attend(ops, u, d, scale=None, window=0, sinks=0, **kw):
    lse = torch.full((u.T, u.Hq), 7.0, device=d["q"].device)
    out = torch.full((u.T, u.Hq, u.hd), 7.0, device=d["q"].device, dtype=u.xd)
    got = ops.paged_attention(u.Hq, u.Hkv, u.hd, u.page, scale, window, sinks)(
        d["q"], d["k"], d["v"], d["table"], d["starts"], d["lens"], out=out, lse=lse, **kw)
    assert got.data_ptr() == out.data_ptr()
    return out, lse


def check_attention(u, out, lse, scale=None, window=0, sinks=0):
    want, wl, weight, size = ref.attention(u, scale, window, sinks)
    used = int(u.starts[-1])
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert (out[used:] == 7.0).all() and (lse[used:] == 7.0).all()          # left as they were
    out, lse, want, wl, weight, size = (x[:used] for x in (out, lse, want, wl, weight, size))
    nan = np.isnan(want)
    assert (np.isnan(out) == nan).all(), np.argwhere(np.isnan(out) != nan)[:5]
    n = int(u.lens.max(initial=0))
    tol = ref.attention_bound(u, want, weight, size, n, u.xd == BF16)
    fin = np.isfinite(want)
    assert (out[~fin & ~nan] == want[~fin & ~nan]).all()
    err = np.abs(out - want)
    assert (err[fin] <= tol[fin]).all(), (np.argwhere(fin & ~(err <= tol))[:5], np.nanmax(err / tol))
    fin = np.isfinite(wl)
    assert (lse[np.isneginf(wl)] == -np.inf).all() and (np.isnan(lse) == np.isnan(wl)).all()
    lim = (2.0 * (u.hd + 8) * (1.0 + size) + 4.0 * (1.0 + np.abs(np.where(fin, wl, 0))) + n) * 2.0 ** -24
    assert (np.abs(lse - wl)[fin] <= lim[fin]).all(), np.nanmax(np.abs(lse - wl)[fin] / lim[fin])


# (new, length) of the sequences; window, sinks
SEQS = {
    "singles": [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 33), (1, 100)],
    "empty": [(0, 0), (1, 0), (0, 40), (2, 1), (5, 3), (1, 40)],
    "prompts": [(37, 37), (1, 1), (64, 64), (65, 65)],
    "chunks": [(5, 70), (33, 129), (17, 17), (2, 64)],
    "long_step": [(1, 2500), (1, 700)],
    "long_chunk": [(70, 1300), (3, 900)],
}
WINDOWS = [(0, 0), (1, 0), (16, 3), (50, 20), (33, 500), (4000, 4)]
LAYOUTS = [(16, 8, 128, 16), (4, 2, 16, 16), (12, 4, 64, 48), (16, 1, 32, 64), (3, 3, 128, 32), (10, 2, 64, 128)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("seqs", SEQS)
def test_attention_shapes(ops, hip_device, seqs, types):
    xd, kd = TYPES[types]
    for i, (hq, hkv, hd, page) in enumerate(LAYOUTS):
        if seqs.startswith("long") and i not in (0, 2):
            continue
        u = Setup(SEQS[seqs], hq, hkv, hd, page, xd, kd, pad=i % 3, seed=i)
        check_attention(u, *attend(ops, u, u.on(hip_device)))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_attention_windows(ops, hip_device, window, sinks, types):
    xd, kd = TYPES[types]
    for name, (hq, hkv, hd, page) in zip(SEQS, LAYOUTS):
        if name == "long_chunk" and window == 4000:
            continue
        u = Setup(SEQS[name], hq, hkv, hd, page, xd, kd, pad=1, seed=window)
        check_attention(u, *attend(ops, u, u.on(hip_device), None, window, sinks), None, window, sinks)


@pytest.mark.parametrize("scale", [1e-3, 0.5, 3.0])
def test_attention_scale(ops, hip_device, scale):
    u = Setup(SEQS["chunks"], 4, 2, 64, 32, F32, BF16, seed=3)
    check_attention(u, *attend(ops, u, u.on(hip_device), scale), scale)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("seqs", ["chunks", "long_chunk", "long_step"])
def test_attention_large_groups_and_many_rows(ops, hip_device, seqs, types):
    """A group of 32 heads on one key head, and chunks over several row tiles."""
    xd, kd = TYPES[types]
    u = Setup(SEQS[seqs], 32, 1, 128, 16, xd, kd, seed=5)
    check_attention(u, *attend(ops, u, u.on(hip_device)))
    u = Setup([(200, 200), (140, 333), (129, 129)], 4, 2, 128, 64, xd, kd, seed=6)
    check_attention(u, *attend(ops, u, u.on(hip_device), None, 60, 7), None, 60, 7)
    check_attention(u, *attend(ops, u, u.on(hip_device)))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("seqs,hq,hkv,hd,page", [
    ([(1, 8300), (1, 1100)] + [(1, 3 + i) for i in range(30)], 8, 8, 32, 64),   # workgroups of 8 waves, no cuts, long walks
    ([(1, 5000), (1, 3)], 4, 2, 64, 16),                                        # more than 16 cuts of a token's keys
    ([(130, 5000)], 64, 64, 32, 128),                                           # long walks of a chunk's tiles
    ([(12, 600), (5, 70)], 6, 2, 64, 16),                                       # 32 rows per workgroup
])
def test_attention_long_walks(ops, hip_device, seqs, hq, hkv, hd, page, types):
    xd, kd = TYPES[types]
    u = Setup(seqs, hq, hkv, hd, page, xd, kd, seed=8)
    d = u.on(hip_device)
    check_attention(u, *attend(ops, u, d))
    if len(seqs) > 1:
        check_attention(u, *attend(ops, u, d, None, 2100, 40), None, 2100, 40)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("case", [0, 1])
def test_attention_many_heads(ops, hip_device, case, hd, types):
    """Row tiles of 32 and 128, with windows, pages that are none and slots that no row sees."""
    seqs, heads, width, _ = ref.MANY_HEADS[case]
    xd, kd = TYPES[types]
    u = Setup(seqs, heads, heads, hd, 16, xd, kd, width=width, pad=1, seed=7)
    d = u.on(hip_device)
    for window, sinks in ((0, 0), (30, 5), (1, 0), (100, 40)):
        check_attention(u, *attend(ops, u, d, None, window, sinks), None, window, sinks)
    u.table[0, 2], u.table[1, 1], u.table[2, -1] = -1, u.n_pages, 2 ** 31 - 1
    for pool in (u.k, u.v):                         # slots past the lengths, and before the second's window
        for s, (_, length) in enumerate(seqs):
            for j in [*range(length, width * 16), *((37,) if s == 1 else ())]:
                if 0 <= u.table[s, j // 16] < u.n_pages:
                    pool[u.table[s, j // 16], :, j % 16] = float("inf") if j % 2 else float("nan")
    d = u.on(hip_device)
    check_attention(u, *attend(ops, u, d, None, 50, 16), None, 50, 16)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("hd", [16, 64, 128])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_attention_unseen_slots_do_not_matter(ops, hip_device, what, hd, types):
    """Slots past a length, before a window and of later tokens of the same
    chunk hold NaN or infinities: rows that do not see them are what they are without them."""
    xd, kd = TYPES[types]
    for seqs, window, sinks, width in (([(9, 40), (1, 21), (150, 150)], 0, 0, 14), ([(9, 90), (1, 130), (140, 200)], 30, 5, 14),
                                       ([(3, 900), (1, 700)], 0, 0, 60), ([(60, 1200), (40, 900)], 0, 0, 80)):
        u = Setup(seqs, 4, 2, hd, 16, xd, kd, width=width, seed=9)
        for s, (n, length) in enumerate(seqs):
            for j in range(width * 16):
                e = u.table[s, j // 16]
                first = length - n
                if j >= length or (window and sinks <= j <= first - window):
                    u.k[e, :, j % 16] = what
                    u.v[e, :, j % 16] = what
            j = length - max(1, n // 2)             # a token of the chunk: those before it do not see it
            u.v[u.table[s, j // 16], 0, j % 16, 3] = what
            u.k[u.table[s, (length - 1) // 16], 1, (length - 1) % 16] = what
        d = u.on(hip_device)
        out, lse = attend(ops, u, d, None, window, sinks)
        want, _, weight, size = ref.attention(u, None, window, sinks)
        got, used = out.double().cpu().numpy(), int(u.starts[-1])
        fin = np.isfinite(want[:used])
        assert fin.any() and not fin.all()
        tol = ref.attention_bound(u, want, weight, np.where(np.isfinite(size), size, 0), 16 * width, xd == BF16)[:used]
        assert (np.isfinite(got[:used]) == fin).all(), np.argwhere(np.isfinite(got[:used]) != fin)[:5]
        assert (np.abs(got[:used] - want[:used])[fin] <= tol[fin]).all()


@pytest.mark.parametrize("types", TYPES)
def test_attention_pages_that_are_none(ops, hip_device, types):
    """Entries outside the pool: NaN for the rows that see a key there, nothing for the others
    (pages before a window, past the length)."""
    xd, kd = TYPES[types]
    u = Setup([(40, 200), (1, 150), (130, 130)], 4, 2, 64, 16, xd, kd, width=16, seed=11)
    u.table[:, 13:] = -1
    u.table[0, 1] = u.n_pages
    u.table[1, 3] = -7
    u.table[2, 4] = 2 ** 31 - 1
    d = u.on(hip_device)
    check_attention(u, *attend(ops, u, d, None, 20, 0), None, 20, 0)
    check_attention(u, *attend(ops, u, d, None, 0, 0))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("hd", [16, 64])
@pytest.mark.parametrize("seqs,heads", [
    ([(1, 48), (1, 30), (1, 48), (2, 17)], (4, 2)),
    ([(30, 48), (9, 30), (48, 48), (2, 17)], (4, 2)),
    ([(1, 3200), (3, 900)], (4, 2)),                                            # in cuts
    ([(150, 208), (40, 200), (208, 208), (9, 90)], (64, 64)),
])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
def test_lengths_past_the_table(ops, hip_device, window, sinks, seqs, heads, hd, types):
    """Sequences 0 and 2 step past their tables: their tokens are not stored and come out as NaN, what the
    cache and its accounts hold stays, and the other sequences do not notice."""
    xd, kd = TYPES[types]
    u = Setup(seqs, *heads, hd, 16, xd, kd, seed=97)
    over = torch.zeros(u.T, dtype=torch.bool)
    for s in range(0, u.S, 2):
        over[u.starts[s]: u.starts[s + 1]] = True
    over = over.to(hip_device)
    inv = (1e6 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32)
    at = torch.from_numpy(inv).to(hip_device), torch.arange(u.T, dtype=torch.int32, device=hip_device)

    def run(lens):
        d = u.on(hip_device)
        d["lens"] = torch.tensor(lens, dtype=torch.int32, device=hip_device)
        q = ops.paged_append(*heads, hd, 16, 1e-6)(d["qkv"], None, None, *at, d["starts"], d["lens"], d["table"], d["k"], d["v"],
                                                   mass=d["mass"])
        kept = {n: d[n].clone() for n in ("k", "v", "mass")}
        out, lse = attend(ops, u, d, None, window, sinks)
        mass = ops.paged_attention_mass(*heads, hd, 16, None, window, sinks)(
            d["q"], lse.nan_to_num(0.0), d["k"], d["table"], d["starts"], d["lens"], d["mass"].clone())
        return q, out, lse, mass, kept

    fine = run(u.lens.tolist())
    assert fine[1].isfinite().all()
    for extra in (1, 37, 2 ** 31 - 1):
        lens = [min(n + extra, 2 ** 31 - 1) if s % 2 == 0 else n for s, n in enumerate(u.lens.tolist())]
        q, out, lse, mass, kept = run(lens)
        assert torch.equal(q, fine[0])
        assert out[over].isnan().all() and lse[over].isnan().all()
        assert torch.equal(out[~over], fine[1][~over]) and torch.equal(lse[~over], fine[2][~over])
        d = u.on(hip_device)
        for s in range(u.S):
            e = torch.from_numpy(u.table[s]).long().to(hip_device)
            for n in ("k", "v", "mass"):
                assert torch.equal(kept[n][e], (d[n] if s % 2 == 0 else fine[4][n])[e])
            assert torch.equal(mass[e], (d["mass"] if s % 2 == 0 else fine[3])[e])


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("new", [100, 1000])
def test_prompts_longer_than_the_table(ops, hip_device, new, types):
    u = Setup([(5, 30), (new, new), (3, 64)], 8, 4, 64, 16, *TYPES[types], width=4, seed=99)
    d = u.on(hip_device)
    inv = torch.ones(32, device=hip_device)
    ops.paged_append(8, 4, 64, 16, 1e-6)(d["qkv"], None, None, inv, torch.zeros(u.T, dtype=torch.int32, device=hip_device),
                                         d["starts"], d["lens"], d["table"], d["k"], d["v"], mass=d["mass"])
    for n in ("k", "v", "mass"):
        e = torch.from_numpy(u.table[1]).long()
        assert torch.equal(d[n].cpu()[e], getattr(u, n)[e])
        setattr(u, n, d[n].cpu())
    out, lse = attend(ops, u, d)
    assert out[5: 5 + new].isnan().all() and lse[5: 5 + new].isnan().all()
    mass = ops.paged_attention_mass(8, 4, 64, 16)(d["q"], lse.nan_to_num(0.0), d["k"], d["table"], d["starts"], d["lens"],
                                                  d["mass"].clone())
    assert torch.equal(mass.cpu()[e], u.mass[e])
    for s, (lo, hi) in ((0, (0, 5)), (2, (5 + new, 8 + new))):
        alone = Setup([u.seqs[s]], 8, 4, 64, 16, *TYPES[types], width=4)
        alone.k, alone.v, alone.q, alone.table, alone.n_pages = u.k, u.v, u.q[lo:hi], u.table[s: s + 1], u.n_pages
        check_attention(alone, out[lo:hi], lse[lo:hi])


def test_evict_of_a_length_past_the_table(ops, hip_device):
    u = Setup([(1, 48), (1, 30)], 4, 2, 64, 16, F32, BF16, spare=6, seed=98)
    d = u.on(hip_device)
    d["lens"][0] = 2 ** 31 - 1
    check_evict(u, d, 33, 2, 5, *run_evict(ops, u, d, 33, 2, 5))


def test_attention_rows_that_all_score_nothing(ops, hip_device):
    """Scores of -infinity everywhere are 0 / 0, as the formula says; one other key is enough."""
    u = Setup([(1, 20), (1, 20)], 2, 1, 64, 16, F32, F32, seed=12)
    u.q.abs_()
    for j in range(20):
        u.k[u.table[0, j // 16], 0, j % 16] = -float("inf")
        if j != 7:
            u.k[u.table[1, j // 16], 0, j % 16] = -float("inf")
    out, lse = attend(ops, u, u.on(hip_device))
    assert out[0].isnan().all()
    assert torch.equal(out[1].cpu(), u.v[u.table[1, 0], 0, 7].expand(2, 64))


def test_attention_past_32_bits(ops, hip_device):
    """Pages whose elements and bytes lie past 2^32."""
    n = 8400                                        # pages of 2^19 bf16 elements: 8.8 GB a pool
    u = Setup([(3, 900), (1, 1500)], 16, 8, 128, 512, F32, BF16, seed=13)
    d = u.on(hip_device)
    move = {int(e): n - 1 - i for i, e in enumerate(u.table.reshape(-1))}
    for name in ("k", "v"):
        big = torch.empty(n, 8, 512, 128, device=hip_device, dtype=BF16)
        for e, to in move.items():
            big[to] = d[name][e]
        d[name] = big
    d["table"] = torch.tensor([[move[int(e)] for e in row] for row in u.table], dtype=torch.int32, device=hip_device)
    out, lse = attend(ops, u, d)
    check_attention(u, out, lse)
    mass = torch.zeros(n, 8, 512, device=hip_device)
    ops.paged_attention_mass(16, 8, 128, 512)(d["q"], lse, d["k"], d["table"], d["starts"], d["lens"], mass)
    small = mass[torch.tensor([move.get(e, 0) for e in range(u.n_pages)])].cpu()
    u.mass.zero_()
    want, _ = ref.mass(u, lse.cpu().numpy())
    for e in move:
        assert np.allclose(small[e].numpy(), want[e], rtol=1e-4, atol=1e-7)


def test_attention_table_slices_and_streams(ops, hip_device):
    """Rows of a wider table, and a call on another stream than the tensors'."""
    u = Setup(SEQS["chunks"], 16, 8, 128, 16, F32, BF16, seed=14)
    d = u.on(hip_device)
    wide = torch.full((u.S, u.width + 5), -1, dtype=torch.int32, device=hip_device)
    wide[:, : u.width] = d["table"]
    base, _ = attend(ops, u, d)
    d["table"] = wide[:, : u.width]
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        out, lse = attend(ops, u, d)
    st.synchronize()
    check_attention(u, out, lse)
    assert torch.equal(base, out)


@pytest.mark.parametrize("types,hd,T", [("f32", 16, 65535 * 32 + 2000), ("bf16", 32, 65535 * 128 + 3000)])
def test_attention_of_millions_of_rows(ops, hip_device, types, hd, T):
    """A prompt of more row tiles than a grid takes, with a window: its ends, where launches meet, and
    rows between."""
    xd, kd = TYPES[types]
    window, page = 20, 4096
    n = -(-T // page)
    g = torch.Generator(device=hip_device).manual_seed(17)
    k, v = (torch.randn(n, 1, page, hd, device=hip_device, generator=g).to(kd) for _ in range(2))
    q = torch.randn(T, 1, hd, device=hip_device, generator=g).to(xd)
    i32 = dict(dtype=torch.int32, device=hip_device)
    table = torch.randperm(n, generator=torch.Generator().manual_seed(18)).to(**i32)[None].contiguous()
    out = torch.full_like(q, float("nan"))
    lse = torch.full((T, 1), float("nan"), device=hip_device)
    ops.paged_attention(1, 1, hd, page, None, window)(q, k, v, table, torch.tensor([0, T], **i32), torch.tensor([T], **i32),
                                                      out=out, lse=lse)
    assert out.isfinite().all() and lse.isfinite().all()
    p = torch.cat([torch.arange(3000), T - 1 - torch.arange(5000), torch.randint(T, (5000,), generator=torch.Generator().manual_seed(19))])
    p = p.to(hip_device)
    j = p[:, None] - torch.arange(window, device=hip_device)
    e = table[0, j.clamp_min(0) // page].long()
    kk, vv = (x[e, 0, j.clamp_min(0) % page].double() for x in (k, v))
    x = (kk * q[p].double()).sum(-1) * hd ** -0.5
    x = x.masked_fill(j < 0, -np.inf)
    want = (torch.softmax(x, -1)[..., None] * vv).sum(1)
    wl = torch.logsumexp(x, -1)
    # scores of at most 30, sums of hd products and 20 keys; 16-bit weights and the output's rounding
    fine = (2.0 * (hd + 8) * 31.0 + 40.0) * 2.0 ** -24 + (2.0 ** -16 if xd == BF16 else 0.0)
    top = vv.abs().amax(1)
    assert ((out[p, 0].double() - want).abs() <= fine * top + HALF_STEP[xd] * (want.abs() + fine * top)).all()
    assert ((lse[p, 0].double() - wl).abs() <= (2.0 * (hd + 8) * 31.0 + 40.0) * 2.0 ** -24).all()


@pytest.mark.parametrize("types", TYPES)
def test_attention_graphs(ops, hip_device, types):
    """Two captured calls with workspaces, replayed in turn with eager calls
    between, on lengths that change under them."""
    xd, kd = TYPES[types]
    u = Setup([(1, 2500), (1, 700)], 16, 8, 128, 64, xd, kd, seed=15)
    d = u.on(hip_device)
    k = ops.paged_attention(16, 8, 128, 64)
    args = (d["k"], d["v"], d["table"], d["starts"], d["lens"])
    q2 = (d["q"].float() * 0.5).to(xd)
    outs = [torch.empty_like(d["q"]) for _ in range(2)]
    k(d["q"], *args, out=outs[0])
    torch.cuda.synchronize()
    graphs = []
    for q, o in ((d["q"], outs[0]), (q2, outs[1])):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            k(q, *args, out=o)
        graphs.append(g)
    for lens in ([2500, 700], [1, 2], [2111, 16], [0, 640]):
        d["lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for q, o in ((d["q"], outs[0]), (q2, outs[1])):
            assert torch.equal(k(q, *args), o)


def test_repeats_bit_for_bit(ops, hip_device):
    for types in TYPES.values():
        u = Setup(SEQS["long_chunk"], 16, 8, 128, 64, *types, seed=16)
        d = u.on(hip_device)
        a, b = attend(ops, u, d), attend(ops, u, d)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        m = [ops.paged_attention_mass(16, 8, 128, 64)(d["q"], a[1], d["k"], d["table"], d["starts"], d["lens"],
                                                      d["mass"].clone()) for _ in range(2)]
        assert torch.equal(*m)


# ------------------------------------------------------------------ append

@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("gains", [True, False])
@pytest.mark.parametrize("seqs", ["singles", "empty", "prompts", "chunks"])
def test_append(ops, hip_device, seqs, gains, types):
    xd, kd = TYPES[types]
    for i, (hq, hkv, hd, page) in enumerate(LAYOUTS):
        u = Setup(SEQS[seqs], hq, hkv, hd, page, xd, kd, pad=i % 3, seed=20 + i)
        if i == 2:
            u.table[0, 0] = -1
            u.table[-1, -1] = u.n_pages
        d = u.on(hip_device)
        pos = u.rng.integers(0, 2 ** 21, u.T).astype(np.int32)
        inv = (1e6 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32)
        gq, gk = [(1 + 0.1 * u.rng.standard_normal(hd)).astype(np.float32) for _ in range(2)] if gains else (None, None)
        want = ref.append(u, gq, gk, inv, pos, 1e-6)
        t = [None if x is None else torch.from_numpy(x).to(hip_device) for x in (gq, gk, inv, pos)]
        keep_mass = i % 2 == 0
        out = torch.full((u.T, hq, hd), 7.0, device=hip_device, dtype=xd)
        ops.paged_append(hq, hkv, hd, page, 1e-6)(d["qkv"], *t, d["starts"], d["lens"], d["table"], d["k"], d["v"],
                                                  mass=d["mass"] if keep_mass else None, out=out)
        used = int(u.starts[-1])
        assert (out[used:] == 7.0).all()
        # the norm's sum of hd squares halves in the root; the rotation adds two products of values of
        # at most the pair's length, angles good to an FP32 rounding; then the stores' own rounding
        x = u.qkv.double().numpy().reshape(u.T, -1, hd)
        size = np.abs(x).max() if not gains else 1.3 * np.sqrt(hd)
        fine = (hd / 2 + 16) * 2.0 ** -24 * 2 * size
        q = out.double().cpu().numpy()[:used]
        assert (np.abs(q - want[0][:used]) <= fine + HALF_STEP[xd] * np.abs(want[0][:used])).all()
        for got, w in ((d["k"], want[1]), (d["v"], want[2])):
            g = got.double().cpu().numpy()
            assert (np.abs(g - w) <= fine + HALF_STEP[kd] * np.abs(w)).all()
        assert np.array_equal(d["mass"].cpu().numpy(), want[3] if keep_mass else u.mass.numpy())


def test_append_angles_far_out(ops, hip_device):
    """Positions up to 2^31 - 1: rotated by the angle's 64-bit product."""
    hd = 128
    u = Setup([(64, 64)], 1, 1, hd, 16, F32, F32, seed=30)
    u.qkv.zero_()
    u.qkv[:, : hd // 2] = 1.0                       # q: the cosines, then the sines
    d = u.on(hip_device)
    pos = np.concatenate((u.rng.integers(0, 2 ** 31, 62), [0, 2 ** 31 - 1])).astype(np.int32)
    inv = (1e6 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32)
    q = ops.paged_append(1, 1, hd, 16, 1e-6)(d["qkv"], None, None, torch.from_numpy(inv).to(hip_device),
                                             torch.from_numpy(pos).to(hip_device), d["starts"], d["lens"], d["table"],
                                             d["k"], d["v"]).double().cpu().numpy()[:, 0]
    ang = pos.astype(np.float64)[:, None] * inv.astype(np.float64)
    # the 64-bit product is off by 2^-53 of up to 2^31, its reduction by as much
    assert np.abs(q[:, : hd // 2] - np.cos(ang)).max() < 4 * 2.0 ** -22 + 2 ** -24
    assert np.abs(q[:, hd // 2:] - np.sin(ang)).max() < 4 * 2.0 ** -22 + 2 ** -24


# ------------------------------------------------------------------ accounts

@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("seqs", SEQS)
def test_mass(ops, hip_device, seqs, types):
    xd, kd = TYPES[types]
    for i, (hq, hkv, hd, page) in enumerate(LAYOUTS):
        if seqs.startswith("long") and i not in (0, 2):
            continue
        window, sinks = WINDOWS[i]
        u = Setup(SEQS[seqs], hq, hkv, hd, page, xd, kd, pad=i % 3, seed=40 + i)
        if seqs == "chunks" and i == 4:
            u.table[1, 2] = -1
        d = u.on(hip_device)
        _, lse = attend(ops, u, d, None, window, sinks)
        lse[~lse.isfinite()] = 0.5                  # rows of the page that is none: any statistics will do
        got = ops.paged_attention_mass(hq, hkv, hd, page, None, window, sinks)(
            d["q"], lse, d["k"], d["table"], d["starts"], d["lens"], d["mass"])
        assert got is d["mass"]
        want, terms = ref.mass(u, lse.cpu().numpy(), None, window, sinks)
        size = hd ** -0.5 * hd * float(u.k.abs().max()) * float(u.q.abs().max()) if hd < 64 else 60.0
        rel = (2.0 * (hd + 8) * (1.0 + size) + 8.0 + terms) * 2.0 ** -24
        assert (np.abs(got.double().cpu().numpy() - want) <= rel * np.abs(want)).all()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5)])
def test_mass_many_rows(ops, hip_device, window, sinks, types):
    """Chunks whose rows are cut over workgroups and joined, beside short ones."""
    xd, kd = TYPES[types]
    u = Setup([(300, 300), (140, 333), (1, 200), (129, 129)], 12, 4, 64, 32, xd, kd, pad=2, seed=45)
    d = u.on(hip_device)
    _, lse = attend(ops, u, d, None, window, sinks)
    got = ops.paged_attention_mass(12, 4, 64, 32, None, window, sinks)(d["q"], lse, d["k"], d["table"], d["starts"],
                                                                       d["lens"], d["mass"])
    want, terms = ref.mass(u, lse.cpu().numpy(), None, window, sinks)
    rel = (2.0 * (64 + 8) * (1.0 + 60.0) + 8.0 + terms) * 2.0 ** -24
    assert (np.abs(got.double().cpu().numpy() - want) <= rel * np.abs(want)).all()


def test_mass_window_at_the_end_of_millions(ops, hip_device):
    """A window far from most keys, under a group whose rows times slots pass 2^31: keys
    that no row sees are left at once and unchanged."""
    g = torch.Generator().manual_seed(51)
    H, page, width, window = 384, 16, 65535 * 8, 40
    q = torch.randn(1, H, 16, generator=g, dtype=torch.float64).float()
    k = torch.randn(5, 1, page, 16, generator=g, dtype=torch.float64).float()
    lse = torch.rand(1, H, generator=g) + 1.0
    table = torch.full((1, width), -1, dtype=torch.int32)
    table[0, -4:] = torch.tensor([3, 0, 4, 1])
    mass = torch.full((5, 1, page), 2.0)
    i32 = dict(dtype=torch.int32, device=hip_device)
    got = ops.paged_attention_mass(H, 1, 16, page, None, window)(
        q.to(hip_device), lse.to(hip_device), k.to(hip_device), table.to(hip_device), torch.tensor([0, 1], **i32),
        torch.tensor([width * page], **i32), mass.to(hip_device)).cpu().double()
    keys = k[[3, 0, 4, 1], 0].reshape(64, 16).double()
    add = torch.exp(0.25 * q[0].double() @ keys.T - lse[0].double()[:, None]).sum(0)
    add[: 64 - window] = 0.0
    want = mass.double()
    want[[3, 0, 4, 1], 0] += add.reshape(4, 16)
    # 384 sums in one lane's order, and exponents below 32 off by 24 steps
    assert torch.allclose(got, want, rtol=(384 + 2 * 24 * 32) * 2.0 ** -24, atol=0.0)
    assert torch.equal(got[2], mass[2].double())


def test_mass_unseen_slots_do_not_matter(ops, hip_device):
    u = Setup([(9, 40), (1, 21)], 4, 2, 64, 16, F32, BF16, width=5, seed=50)
    for s, (_, length) in enumerate(u.seqs):
        for j in range(length, 80):
            u.k[u.table[s, j // 16], :, j % 16] = float("nan")
            u.mass[u.table[s, j // 16], :, j % 16] = 3.0
    d = u.on(hip_device)
    _, lse = attend(ops, u, d)
    got = ops.paged_attention_mass(4, 2, 64, 16)(d["q"], lse, d["k"], d["table"], d["starts"], d["lens"], d["mass"])
    want, _ = ref.mass(u, lse.cpu().numpy())
    assert np.allclose(got.cpu().numpy(), want, rtol=1e-4)


# ------------------------------------------------------------------ eviction

def run_evict(ops, u, d, keep, sinks, recent):
    tw = -(-keep // u.page)
    to = torch.from_numpy(u.free[: u.S * tw].reshape(u.S, tw).copy()).to(d["k"].device)
    lens, kept = ops.paged_evict(u.Hkv, u.hd, u.page, keep, sinks, recent)(d["k"], d["v"], d["mass"], d["table"],
                                                                          d["lens"], to)
    return lens, kept, to


def check_evict(u, d, keep, sinks, recent, lens, kept, to):
    wl, wk = ref.evict(u, keep, sinks, recent)
    assert np.array_equal(lens.cpu().numpy(), wl)
    assert np.array_equal(kept.cpu().numpy(), wk)
    want = {n: getattr(u, n).clone() for n in ("k", "v", "mass")}
    to = to.cpu().numpy()
    for s in range(u.S):
        for h in range(u.Hkv):
            for i in range(int(wl[s])):
                j = int(wk[s, h, i])
                a, b = int(u.table[s, j // u.page]), int(to[s, i // u.page])
                if not 0 <= b < u.n_pages:
                    continue
                for n, w in want.items():
                    ok = 0 <= a < u.n_pages
                    w[b, h, i % u.page] = getattr(u, n)[a, h, j % u.page] if ok else float("nan")
    for n, w in want.items():
        assert torch.equal(torch.nan_to_num(d[n].cpu(), 9.0), torch.nan_to_num(w, 9.0)), n
        assert torch.equal(d[n].cpu().isnan(), w.isnan()), n


@pytest.mark.parametrize("kd", [F32, BF16])
@pytest.mark.parametrize("hd,page", [(16, 16), (32, 48), (64, 16), (128, 64)])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (7, 3, 4), (40, 4, 16), (64, 0, 0), (100, 0, 100), (300, 5, 9)])
def test_evict(ops, hip_device, keep, sinks, recent, hd, page, kd):
    u = Setup([(1, 0), (1, 1), (1, 39), (1, 64), (1, 150), (1, 251)], 4, 2, hd, page, F32, kd,
              spare=6 * -(-keep // page), seed=60)
    u.mass[u.mass < 0.5] = 0.0                      # many ties
    u.mass[u.table[4, 0], 0, 5] = float("nan")
    u.mass[u.table[4, 0], 1, 9] = -float("nan")
    u.mass[u.table[5, 0], 0, 6] = float("inf")
    u.mass[u.table[5, 0], 1] = -0.0
    u.mass[u.table[5, 0], 1, 3] = -1.0
    d = u.on(hip_device)
    check_evict(u, d, keep, sinks, recent, *run_evict(ops, u, d, keep, sinks, recent))


@pytest.mark.parametrize("length", [3000, 9000, 20000, 40000, 70001])
def test_evict_lengths(ops, hip_device, length):
    """Every way the ranks are held, with all weights the same and with few values."""
    keep = length // 3
    for few in (False, True):
        u = Setup([(1, length)], 1, 1, 16, 64, F32, F32, spare=-(-keep // 64), seed=61)
        u.mass = torch.full_like(u.mass, 0.25) if few else (u.mass * 4).floor()
        d = u.on(hip_device)
        lens, kept, to = run_evict(ops, u, d, keep, 4, 50)
        _, want = ref.evict(u, keep, 4, 50)
        assert np.array_equal(kept.cpu().numpy(), want)
        j = kept[0, 0].long()
        rows = lambda pool, t: pool[t[0].long(), 0].flatten(0, 1)   # noqa: E731
        for n in ("k", "v", "mass"):
            assert torch.equal(rows(d[n], to)[:keep], rows(d[n], d["table"])[j])


def test_evict_pages_that_are_none(ops, hip_device):
    u = Setup([(1, 60), (1, 100)], 4, 2, 64, 16, F32, F32, spare=8, seed=62)
    u.table[0, 1] = -1
    u.table[1, 6] = u.n_pages
    u.free[5] = -1
    u.free[2] = u.n_pages
    d = u.on(hip_device)
    check_evict(u, d, 50, 2, 5, *run_evict(ops, u, d, 50, 2, 5))


def test_evict_shared_pages(ops, hip_device):
    """Two sequences share a prompt's pages; each moves to pages of its own, the
    shared ones stay as they are."""
    u = Setup([(1, 64), (1, 60)], 4, 2, 64, 16, F32, BF16, spare=8, seed=63)
    u.table[1, :2] = u.table[0, :2]
    d = u.on(hip_device)
    check_evict(u, d, 33, 2, 5, *run_evict(ops, u, d, 33, 2, 5))


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("types", TYPES)
def test_run_of_all(ops, hip_device, types):
    """A prompt in two chunks, accounts, eviction, then tokens one by one with a
    window, as a program would; each step against the formulas on the state it found."""
    xd, kd = TYPES[types]
    hq, hkv, hd, page, S = 8, 4, 64, 16, 3
    u = Setup([(n, n) for n in (70, 33, 50)], hq, hkv, hd, page, xd, kd, width=6, spare=S * 3 + 2, seed=70)
    dev = hip_device
    d = u.on(dev)
    inv = torch.from_numpy((1e6 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32)).to(dev)
    gains = [torch.ones(hd, device=dev) for _ in range(2)]
    app, pos = ops.paged_append(hq, hkv, hd, page, 1e-6), np.zeros(S, np.int64)

    def step(new, lens, table, window=0, sinks=0):
        u.seqs = list(zip(new, lens))
        u.starts = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
        u.lens, u.T = np.array(lens, np.int32), int(sum(new))
        u.table = table.cpu().numpy()
        u.width = u.table.shape[1]
        g = torch.Generator().manual_seed(int(pos.sum()))
        qkv = torch.randn(u.T, (hq + 2 * hkv) * hd, generator=g).to(xd)
        p = np.concatenate([pos[s] + np.arange(new[s]) for s in range(S)]).astype(np.int32)
        pos[:] += new
        starts, ln = torch.from_numpy(u.starts).to(dev), torch.from_numpy(u.lens).to(dev)
        q = app(qkv.to(dev), *gains, inv, torch.from_numpy(p).to(dev), starts, ln, table, d["k"], d["v"], mass=d["mass"])
        lse = torch.empty(u.T, hq, device=dev)
        out = ops.paged_attention(hq, hkv, hd, page, None, window, sinks)(q, d["k"], d["v"], table, starts, ln, lse=lse)
        u.q, u.k, u.v, u.mass = q.cpu(), d["k"].cpu(), d["v"].cpu(), d["mass"].cpu()
        check_attention(u, out, lse, None, window, sinks)
        ops.paged_attention_mass(hq, hkv, hd, page, None, window, sinks)(q, lse, d["k"], table, starts, ln, d["mass"])
        want, _ = ref.mass(u, lse.cpu().numpy(), None, window, sinks)
        assert np.allclose(d["mass"].cpu().numpy(), want, rtol=2e-4, atol=0)
        u.mass = d["mass"].cpu()

    lens = [30, 33, 20]
    step(lens, lens, d["table"])
    step([40, 0, 30], [70, 33, 50], d["table"])
    to = torch.from_numpy(u.free[: S * 3].reshape(S, 3).copy()).to(dev)
    new_lens, kept = ops.paged_evict(hkv, hd, page, 40, 4, 8)(d["k"], d["v"], d["mass"], d["table"],
                                                              torch.from_numpy(u.lens).to(dev), to)
    check_evict(u, d, 40, 4, 8, new_lens, kept, to)
    lens = new_lens.tolist()
    for i in range(3):
        lens = [n + 1 for n in lens]
        step([1] * S, lens, to, window=0 if i else 20, sinks=0 if i else 4)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("n", [1, 30])
def test_more_sequences_than_lanes(ops, hip_device, n, types):
    """150 sequences, some without new tokens and some empty, ends and starts of 64 among them."""
    xd, kd = TYPES[types]
    rng = np.random.default_rng(95)
    seqs = [(0, 0) if s % 17 == 3 else (0, 20) if s % 13 == 5 else (k := int(rng.integers(1, 2 * n + 1)),
                                                                   k + int(rng.integers(0, 50))) for s in range(150)]
    for s in (62, 63, 64, 65, 127, 128, 149):
        seqs[s] = (n, n + 7) if s % 2 else (0, 9)
    u = Setup(seqs, 8, 2, 32, 16, xd, kd, pad=3, seed=96)
    d = u.on(hip_device)
    out, lse = attend(ops, u, d)
    check_attention(u, out, lse)
    mass = ops.paged_attention_mass(8, 2, 32, 16)(d["q"], lse, d["k"], d["table"], d["starts"], d["lens"], d["mass"].clone())
    want, terms = ref.mass(u, lse.cpu().numpy())
    size = 32 ** 0.5 * float(u.k.abs().max()) * float(u.q.abs().max())
    rel = (2.0 * (32 + 8) * (1.0 + size) + 8.0 + terms) * 2.0 ** -24
    assert (np.abs(mass.double().cpu().numpy() - want) <= rel * np.abs(want)).all()
    inv = (1e6 ** (-np.arange(0, 32, 2) / 32)).astype(np.float32)
    pos = rng.integers(0, 2 ** 21, u.T).astype(np.int32)
    want = ref.append(u, None, None, inv, pos, 1e-6)
    q = ops.paged_append(8, 2, 32, 16, 1e-6)(d["qkv"], None, None, torch.from_numpy(inv).to(hip_device),
                                             torch.from_numpy(pos).to(hip_device), d["starts"], d["lens"], d["table"],
                                             d["k"], d["v"], mass=d["mass"])
    used = int(u.starts[-1])
    fine = (32 / 2 + 16) * 2.0 ** -24 * 2 * float(u.qkv.abs().max())
    for got, w, t in ((q[:used], want[0][:used], xd), (d["k"], want[1], kd), (d["v"], want[2], kd)):
        assert (np.abs(got.double().cpu().numpy() - w) <= fine + HALF_STEP[t] * np.abs(w)).all()
    assert np.array_equal(d["mass"].cpu().numpy(), want[3])


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("new", [1, 180])
def test_run_captured(ops, hip_device, types, new):
    """Append, attention, accounts and the lengths' step in one graph, and eviction in another,
    replayed on new contents with eager runs of the same between: equal bit for bit."""
    xd, kd = TYPES[types]
    hq, hkv, hd, page, S, keep = 8, 2, 128, 64, 2, 300
    u = Setup([(new, 700)] * S, hq, hkv, hd, page, xd, kd, width=22, spare=S * 5, seed=80)
    inv = torch.from_numpy((1e6 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32)).to(hip_device)
    to = torch.from_numpy(u.free[: S * 5].reshape(S, 5).copy()).to(hip_device)
    app, att = ops.paged_append(hq, hkv, hd, page, 1e-6), ops.paged_attention(hq, hkv, hd, page)
    acc, evi = ops.paged_attention_mass(hq, hkv, hd, page), ops.paged_evict(hkv, hd, page, keep, 4, 16)

    def state():
        d = u.on(hip_device)
        d["pos"] = torch.arange(u.T, dtype=torch.int32, device=hip_device) % new + 700 - new
        d["lse"] = torch.zeros(u.T, hq, device=hip_device)
        return d

    def step(d):
        q = app(d["qkv"], None, None, inv, d["pos"], d["starts"], d["lens"], d["table"], d["k"], d["v"], mass=d["mass"])
        out = att(q, d["k"], d["v"], d["table"], d["starts"], d["lens"], lse=d["lse"])
        acc(q, d["lse"], d["k"], d["table"], d["starts"], d["lens"], d["mass"])
        d["lens"].add_(new)
        d["pos"].add_(new)
        return q, out

    def cut(d):
        return evi(d["k"], d["v"], d["mass"], d["table"], d["lens"], to)

    a, b = state(), state()
    for f in (step, cut):                           # on a state of their own: kernels loaded before they are captured
        f(state())
    torch.cuda.synchronize()
    graphs, outs = [], []
    for f in (step, cut):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(f(b))
        graphs.append(g)
    g = torch.Generator().manual_seed(81)
    for _ in range(3):
        x = torch.randn(u.T, (hq + 2 * hkv) * hd, generator=g).to(xd).to(hip_device)
        for d in (a, b):
            d["qkv"].copy_(x)
        graphs[0].replay()
        want = step(a)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, outs[0]))
        graphs[1].replay()
        want = cut(a)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, outs[1]))
        assert all(torch.equal(a[n], b[n]) for n in ("k", "v", "mass", "lens", "lse"))
        assert want[0].tolist() == [keep] * S


def test_calls_on_two_streams_at_once(ops, hip_device):
    """Calls with workspaces of their own, interleaved on two streams."""
    runs = []
    for seed, (xd, kd) in enumerate(TYPES.values()):
        u = Setup([(1, 2900), (40, 1300)], 16, 8, 128, 64, xd, kd, seed=90 + seed)
        d = u.on(hip_device)
        out, lse = attend(ops, u, d)
        mass = ops.paged_attention_mass(16, 8, 128, 64)(d["q"], lse, d["k"], d["table"], d["starts"], d["lens"],
                                                        d["mass"].clone())
        runs.append((u, d, out, lse, mass))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(12):
        u, d, _, lse, _ = runs[i % 3]
        with torch.cuda.stream(streams[i % 2]):
            got.append((*attend(ops, u, d), ops.paged_attention_mass(16, 8, 128, 64)(
                d["q"], lse, d["k"], d["table"], d["starts"], d["lens"], d["mass"].clone())))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(x, runs[i % 3][2:]))


def test_trunk_layers_from_operators(ops, hip_device):
    """The tiny trunk driven through the operator API on a paged cache gives the
    hidden state of the engine's prefill, prompt in chunks included."""
    from oracle.model import Shape, synthetic_weights
    from soraku_amd import GraphFrameEngine
    from soraku_amd.config import TINY

    sh = Shape(**{k: getattr(TINY, k) for k in ("d_model", "n_layers", "n_q_heads", "n_kv_heads", "head_dim",
                                               "trunk_inter", "depth_mult", "n_codebooks", "codebook_size", "text_vocab")})
    w = synthetic_weights(sh, 5)
    rng = np.random.default_rng(5)
    text, prompt = rng.integers(0, TINY.text_vocab, 21), rng.integers(0, TINY.codebook_size, (12, TINY.n_codebooks))
    e = GraphFrameEngine(device="cuda:0", max_cache_len=64, cfg_scale=1.0, batch=1, state_dict=w, shape=TINY)
    want = e.prefill(text, None, prompt).cpu().numpy()[0]
    e.close()
    t = {k: torch.as_tensor(np.asarray(v)).to(hip_device).float().contiguous() for k, v in w.items()}
    frames = np.concatenate((np.full((1, TINY.n_codebooks), TINY.bos_id), prompt))
    x = torch.cat([t["trunk.embed_tokens.weight"][torch.from_numpy(text).to(hip_device)],
                   ops.frame_embed(len(frames), TINY.n_codebooks, TINY.audio_vocab, TINY.d_model, TINY.frame_scale)(
                       torch.from_numpy(frames).to(hip_device), t["audio_codebooks.table"])])
    D, I, hq, hkv, hd, page = TINY.d_model, TINY.trunk_inter, TINY.n_q_heads, TINY.n_kv_heads, TINY.head_dim, 16
    nq = (hq + 2 * hkv) * hd
    pools = [(torch.zeros(5, hkv, page, hd, device=hip_device), torch.zeros(5, hkv, page, hd, device=hip_device))
             for _ in range(TINY.n_layers)]
    table = torch.tensor([[4, 0, 2]], dtype=torch.int32, device=hip_device)
    inv = torch.from_numpy((TINY.rope_theta ** (-np.arange(0, hd, 2) / hd)).astype(np.float32)).to(hip_device)
    zero = torch.zeros(max(nq, D), device=hip_device)
    done = 0
    for n in (1, 20, 13):                           # 34 tokens in three chunks
        y = x[done: done + n].contiguous()
        done += n
        starts, lens = (torch.tensor(v, dtype=torch.int32, device=hip_device) for v in ([0, n], [done]))
        pos = torch.arange(done - n, done, dtype=torch.int32, device=hip_device)
        for i in range(TINY.n_layers):
            L = f"trunk.layers.{i}."
            a = ops.rmsnorm(n, D, TINY.trunk_eps)(y, t[L + "input_layernorm.weight"])
            wqkv = torch.cat([t[L + f"self_attn.{p}_proj.weight"] for p in "qkv"]).contiguous()
            qkv = ops.classifier_gemv(n, nq, D)(a, wqkv, zero[:nq])
            q = ops.paged_append(hq, hkv, hd, page, TINY.trunk_eps)(
                qkv, t[L + "self_attn.q_norm.weight"], t[L + "self_attn.k_norm.weight"], inv, pos, starts, lens, table, *pools[i])
            o = ops.paged_attention(hq, hkv, hd, page)(q, *pools[i], table, starts, lens)
            y = ops.down_residual_gemv(n, D, hq * hd)(o.view(n, hq * hd), t[L + "self_attn.o_proj.weight"], y)
            a = ops.rmsnorm(n, D, TINY.trunk_eps)(y, t[L + "post_attention_layernorm.weight"])
            act = ops.swiglu_gemv(n, I, D)(a, t[L + "mlp.gate_proj.weight"], t[L + "mlp.up_proj.weight"])
            y = ops.down_residual_gemv(n, D, I)(act, t[L + "mlp.down_proj.weight"], y)
        got = ops.rmsnorm(n, D, TINY.trunk_eps)(y, t["trunk.norm.weight"])[-1].cpu().numpy()
    assert done == len(x)
    # 2 layers of FP32 sums of up to 128 terms, in other orders
    assert np.abs(got - want).max() <= 2e-5 * np.abs(want).max()


def test_engine_cache_as_pages(ops, hip_device):
    """An engine's cache is a pool with one page per row."""
    import ctypes as C

    from oracle.model import Shape, synthetic_weights
    from soraku_amd import GraphFrameEngine
    from soraku_amd._lib import check, lib
    from soraku_amd.config import TINY

    sh = Shape(**{k: getattr(TINY, k) for k in ("d_model", "n_layers", "n_q_heads", "n_kv_heads", "head_dim",
                                               "trunk_inter", "depth_mult", "n_codebooks", "codebook_size", "text_vocab")})
    rng = np.random.default_rng(6)
    e = GraphFrameEngine(device="cuda:0", max_cache_len=64, cfg_scale=1.5, batch=2, state_dict=synthetic_weights(sh, 6),
                         shape=TINY)
    e.prefill(rng.integers(0, TINY.text_vocab, 30), np.array([1]), None)
    u = Setup([(1, 31), (1, 2)], TINY.n_q_heads, TINY.n_kv_heads, TINY.head_dim, 64, spare=0, seed=80)
    u.table = np.array([[0], [1]], np.int32)
    n = 2 * TINY.n_kv_heads * 64 * TINY.head_dim

    class Wrap:
        def __init__(self, ptr):
            self.__cuda_array_interface__ = {"shape": (2, TINY.n_kv_heads, 64, TINY.head_dim), "typestr": "<f4",
                                             "data": (ptr, False), "version": 3}
    d = u.on(hip_device)
    for kv, name in enumerate(("k", "v")):
        p = C.c_void_p()
        check(lib().sk_kv_ptr(e._h, 1, kv, C.byref(p)))
        d[name] = torch.as_tensor(Wrap(p.value), device=hip_device)
        assert d[name].numel() == n
        setattr(u, name, d[name].cpu())
    check_attention(u, *attend(ops, u, d))
    e.close()
