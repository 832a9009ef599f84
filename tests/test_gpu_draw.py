"""Sampling by row on the GPU against the whole row sorted in 64 bits (draw_ref.py): vocabularies in one workgroup and in
several, every filter, equal and masked values, infinities and NaN, guidance, masks of bits, graphs and streams."""

import numpy as np
import pytest
import torch

import draw_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops(hip_device):
    from soraku_amd import ops as O

    return O


def words_of(mask):
    """Bits [rows, V] as int32 words."""
    pad = np.zeros((mask.shape[0], -(-mask.shape[1] // 32) * 32), bool)
    pad[:, : mask.shape[1]] = mask
    return torch.from_numpy(np.packbits(pad, axis=1, bitorder="little").view(np.int32).copy())


def sample(ops, dev, logits, u, cfg=False, allowed=None, **p):
    rows = logits.shape[0]
    on = {k: None if v is None else torch.as_tensor(v).to(dev) for k, v in p.items()}
    logprob, kept = torch.full((rows,), 7.0, device=dev), torch.full((rows,), -5, device=dev, dtype=torch.int32)
    out = ops.sample_rows(logits.shape[-1], cfg=cfg)(
        logits.to(dev), torch.as_tensor(u, dtype=torch.float64).to(dev), logprob=logprob, kept=kept,
        allowed=None if allowed is None else words_of(allowed).to(dev), **on)
    return out.cpu().numpy(), logprob.double().cpu().numpy(), kept.cpu().numpy()


def check(ops, dev, logits, u, cfg=False, allowed=None, least=0.9, **p):
    """Every row whose draw is determined; at least so many of them are (fewer where weights are equal and a
    bound, p of their number, is a sum of theirs itself)."""
    got, logprob, kept = sample(ops, dev, logits, u, cfg, allowed, **p)
    x = logits.float().numpy()
    if cfg:
        x = ref.merge(x, p["cfg_scale"].numpy())
    sure = 0
    for r in range(len(got)):
        args = {k: float(v[r]) if k != "top_k" else int(v[r]) for k, v in p.items() if v is not None and k != "cfg_scale"}
        a = None if allowed is None else allowed[r if len(allowed) > 1 else 0]
        tok, lp, n, margin, n_sure = ref.row(x[r], float(u[r]), allowed=a, **args)
        if n_sure:
            assert kept[r] == n, (r, kept[r], n, args)
        if n_sure and margin > ref.safe(x.shape[1]):
            sure += 1
            assert got[r] == tok, (r, got[r], tok, margin, args)
            if np.isinf(lp):
                assert logprob[r] == lp
            else:
                # y - y0 and the sum's logarithm in 64 bits, their difference rounded once; sums are within 1e-9
                assert abs(logprob[r] - lp) <= abs(lp) * 2.0 ** -24 + 1e-8, (r, logprob[r], lp)
    assert sure >= least * len(got), sure


def params(rng, rows, **kw):
    """Parameters by row: of each filter some rows have none."""
    out = {}
    f = lambda a: torch.from_numpy(np.asarray(a, np.float32))  # noqa: E731
    if kw.get("temperature", True):
        out["temperature"] = f(rng.choice([0.0, 0.5, 0.8, 1.0, 1.3], rows))
    if kw.get("top_k", True):
        out["top_k"] = torch.from_numpy(rng.choice([0, 1, 2, 50, 400, 10 ** 9, -3], rows).astype(np.int32))
    if kw.get("top_p", True):
        out["top_p"] = f(rng.choice([0.0, 0.01, 0.5, 0.9, 0.95, 0.999999, 1.0, 2.0], rows))
    if kw.get("min_p", True):
        out["min_p"] = f(rng.choice([0.0, 1e-30, 1e-4, 0.02, 0.5, 1.0, 1.5], rows))
    return out


SIZES = [1, 2, 3, 31, 33, 100, 1024, 2051, 5000, 16384, 16385, 40000, 151936]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", SIZES)
def test_sizes(ops, hip_device, v, dtype):
    rng = np.random.default_rng(v)
    for rows, spread in ((1, 2.5), (40 if v > 20000 else 120, 2.5), (7, 8.0)):
        x = torch.from_numpy(rng.standard_normal((rows, v)).astype(np.float32) * np.float32(spread)).to(dtype)
        check(ops, hip_device, x, rng.random(rows), **params(rng, rows))
    check(ops, hip_device, x, rng.random(rows))      # no parameters at all


@pytest.mark.parametrize("only", ["temperature", "top_k", "top_p", "min_p"])
@pytest.mark.parametrize("v", [2051, 30000])
def test_one_filter_at_a_time(ops, hip_device, v, only):
    rng = np.random.default_rng(v + len(only))
    x = torch.from_numpy(rng.standard_normal((64, v)).astype(np.float32) * np.float32(3.0))
    check(ops, hip_device, x, rng.random(64), **{k: w for k, w in params(rng, 64).items() if k == only})


@pytest.mark.parametrize("v", [100, 2051, 20000, 151936])
def test_equal_values(ops, hip_device, v):
    """All equal, two values, a handful of values: more equal ones than any list holds."""
    rng = np.random.default_rng(v)
    rows = 24
    for levels in (1, 2, 5):
        x = torch.from_numpy(rng.integers(0, levels, (rows, v)).astype(np.float32))
        check(ops, hip_device, x, rng.random(rows), least=0.6, **params(rng, rows))
        check(ops, hip_device, -x.to(BF16) * 0.0, rng.random(rows), least=0.6, **params(rng, rows))   # -0 and 0


@pytest.mark.parametrize("v", [2051, 20000, 151936])
def test_close_values(ops, hip_device, v, least=0.9):
    """Values that differ in their last bits only, thousands to a bucket."""
    rng = np.random.default_rng(v + 1)
    rows = 16
    x = (4.0 + rng.integers(0, 5000, (rows, v)) * 2.0 ** -21).astype(np.float32)
    check(ops, hip_device, torch.from_numpy(x), rng.random(rows), least=least, **params(rng, rows))


@pytest.mark.parametrize("v", [64, 2051, 20000, 151936])
def test_masked_and_infinite_values(ops, hip_device, v):
    """Rows of which little or nothing is left: -inf, the type's lowest value, NaN, +inf, and rows of those alone."""
    rng = np.random.default_rng(v + 2)
    low = torch.finfo(F32).min
    x = torch.from_numpy(rng.standard_normal((16, v)).astype(np.float32) * np.float32(2.0))
    hide = torch.from_numpy(rng.random((16, v)) < 0.999)
    x[0] = -float("inf")
    x[1] = float("nan")
    x[2] = low
    x[3][hide[3]] = -float("inf")
    x[4][hide[4]] = low
    x[5][hide[5]] = float("nan")
    x[6, 5] = float("inf")
    x[7, :3] = torch.tensor([float("nan"), float("inf"), -float("inf")])
    x[8] = -float("inf")
    x[8, v - 1] = 1.0
    x[9] = low
    x[9, v // 2] = -1e30
    x[10][hide[10]] = -1e30
    x[11] = x[11] * 1e36
    x[12] = x[12] * 1e-40
    x[13] = float("inf")
    x[14, v // 3:] = -10000.0
    x[15] = torch.finfo(F32).max
    for _ in range(3):
        check(ops, hip_device, x, rng.random(16), least=0.6, **params(rng, 16))
    check(ops, hip_device, x, rng.random(16))


@pytest.mark.parametrize("v", [500, 20000])
@pytest.mark.parametrize("temp", [1e-38, 1e-30, 1e-12, 1e-4, 100.0, 1e30, float("inf"), float("nan"), -1.0])
def test_temperatures(ops, hip_device, v, temp):
    rng = np.random.default_rng(7)
    x = torch.from_numpy(rng.standard_normal((8, v)).astype(np.float32) * np.float32(4.0))
    p = params(rng, 8, top_k=False)
    p["temperature"] = torch.full((8,), temp)
    check(ops, hip_device, x, rng.random(8), least=0.6, **p)


@pytest.mark.parametrize("v", [77, 20000])
def test_ends_of_the_draw(ops, hip_device, v):
    """u of 0 and the last number below 1, and past them: the first and the last kept one."""
    rng = np.random.default_rng(v)
    x = torch.from_numpy(rng.standard_normal((6, v)).astype(np.float32))
    u = np.array([0.0, 1 - 2.0 ** -53, 1.0, 2.0, -1.0, np.nan])
    for p in ({}, dict(top_k=torch.full((6,), 9, dtype=torch.int32)), dict(top_p=torch.full((6,), 0.3)), dict(min_p=torch.full((6,), 0.4))):
        got, logprob, kept = sample(ops, hip_device, x, u, **p)
        for r in range(6):
            args = {k: float(t[r]) if k != "top_k" else int(t[r]) for k, t in p.items()}
            first, _, n, _, _ = ref.row(x[r].numpy(), 0.0, **args)
            last, _, _, _, _ = ref.row(x[r].numpy(), 1.0, **args)
            assert kept[r] == n and got[r] == (first if r in (0, 4, 5) else last)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [40, 2051, 20000])
def test_guidance_and_allowed(ops, hip_device, v, dtype):
    rng = np.random.default_rng(v + 5)
    rows = 48
    x = torch.from_numpy(rng.standard_normal((rows, 2, v)).astype(np.float32) * np.float32(2.0)).to(dtype)
    x[3, 1, 4], x[4, 0, 4] = float("inf"), float("nan")
    scale = torch.from_numpy(rng.uniform(0.0, 3.0, rows).astype(np.float32))
    scale[0], scale[1], scale[2] = 0.0, 1.0, -1.5
    allowed = rng.random((rows, v)) < 0.7
    allowed[5] = False
    allowed[6] = False
    allowed[6, v - 1] = True
    check(ops, hip_device, x, rng.random(rows), cfg=True, cfg_scale=scale, **params(rng, rows))
    check(ops, hip_device, x, rng.random(rows), cfg=True, allowed=allowed, cfg_scale=scale, **params(rng, rows))
    check(ops, hip_device, x[:, 0].contiguous(), rng.random(rows), allowed=allowed, **params(rng, rows))
    check(ops, hip_device, x[:, 0].contiguous(), rng.random(rows), allowed=allowed[:1], **params(rng, rows))


def test_the_engine_s_sampler_agrees(ops, hip_device):
    """The same codes as the operator for one utterance, with guidance and blocked ids."""
    rng = np.random.default_rng(11)
    rows, v = 60, 2051
    x = torch.from_numpy(rng.standard_normal((rows, 2, v)).astype(np.float32) * np.float32(2.0)).to(hip_device)
    u = rng.random(rows)
    allowed = np.ones((1, v), bool)
    allowed[0, [2048, 2049, 2050]] = False
    one = ops.sample(v, 2048, 2049, 2050)
    want = [int(one(x[r], cfg_scale=1.5, q=3, mask_eos_q0=False, temperature=0.9, top_k=50, top_p=0.95, u=u[r])) for r in range(rows)]
    full = lambda c, t=F32: torch.full((rows,), c, device=hip_device, dtype=t)  # noqa: E731
    got = ops.sample_rows(v, cfg=True)(x, torch.from_numpy(u).to(hip_device), temperature=full(0.9), top_k=full(50, torch.int32),
                                       top_p=full(0.95), cfg_scale=full(1.5), allowed=words_of(allowed).to(hip_device))
    assert got.tolist() == want


def test_rows_apart(ops, hip_device):
    """Rows of a wider tensor, as a padded classifier leaves them, and rows of no alignment."""
    rng = np.random.default_rng(12)
    for v, wide, at in ((2051, 2176, 0), (20000, 20011, 3), (33, 40, 7)):
        x = torch.from_numpy(rng.standard_normal((9, wide)).astype(np.float32)).to(hip_device)
        u = torch.from_numpy(rng.random(9)).to(hip_device)
        f = ops.sample_rows(v)
        assert torch.equal(f(x[:, at: at + v], u), f(x[:, at: at + v].contiguous(), u))
        y = x[:8].view(4, 2, wide)[:, :, :v]
        s = torch.ones(4, device=hip_device)
        g = ops.sample_rows(v, cfg=True)
        assert torch.equal(g(y, u[:4], cfg_scale=s), g(y.contiguous(), u[:4], cfg_scale=s))


def test_far_rows(ops, hip_device):
    """Logits past 2^31 elements and 2^32 bytes."""
    rows, v = 15000, 151936
    x = torch.zeros(rows, v, device=hip_device, dtype=BF16)
    ids = torch.randint(0, v, (rows,), generator=torch.Generator().manual_seed(1)).to(hip_device)
    x.scatter_(1, ids[:, None], 90.0)
    u = torch.rand(rows, device=hip_device, dtype=torch.float64) * 0.999
    assert torch.equal(ops.sample_rows(v)(x, u), ids)


def test_largest_vocabulary(ops, hip_device):
    rng = np.random.default_rng(13)
    x = torch.from_numpy(rng.standard_normal((3, 1 << 20)).astype(np.float32) * np.float32(1.5))
    check(ops, hip_device, x, rng.random(3), top_p=torch.tensor([0.5, 0.95, 0.0]))
    check(ops, hip_device, x, rng.random(3), top_k=torch.tensor([50, 4097, 900000], dtype=torch.int32))


def test_no_rows(ops, hip_device):
    u = torch.empty(0, device=hip_device, dtype=torch.float64)
    assert ops.sample_rows(50)(torch.empty(0, 50, device=hip_device), u).shape == (0,)
    assert ops.sample_rows(50, cfg=True)(torch.empty(0, 2, 50, device=hip_device), u, cfg_scale=u.float()).shape == (0,)


def test_repeats_and_batches(ops, hip_device):
    """The same bits again, and for a row alone or among others."""
    rng = np.random.default_rng(14)
    for v in (2051, 151936):
        x = torch.from_numpy(rng.standard_normal((40, v)).astype(np.float32) * np.float32(2.0)).to(hip_device)
        p = {k: t.to(hip_device) for k, t in params(rng, 40).items()}
        u = torch.from_numpy(rng.random(40)).to(hip_device)
        f = ops.sample_rows(v)

        def run(s):
            lp = torch.empty(len(u[s]), device=hip_device)
            return f(x[s], u[s], logprob=lp, **{k: t[s] for k, t in p.items()}), lp
        tok, lp = run(slice(0, 40))
        for s in (slice(0, 40), slice(3, 4), slice(10, 30)):
            t2, l2 = run(s)
            assert torch.equal(t2, tok[s])
            # sums over other slices may be a few 2^-44 apart
            assert torch.equal(l2.isinf(), lp[s].isinf()) and torch.allclose(l2, lp[s], rtol=2.0 ** -23, atol=1e-9)


@pytest.mark.parametrize("v", [2051, 50000])
def test_captured_and_replayed(ops, hip_device, v):
    """Parameters and draws are read when the graph runs."""
    rng = np.random.default_rng(v)
    rows = 6
    x = torch.empty(rows, v, device=hip_device)
    u = torch.zeros(rows, device=hip_device, dtype=torch.float64)
    p = {k: t.to(hip_device) for k, t in params(rng, rows).items()}
    out = torch.empty(rows, device=hip_device, dtype=torch.int64)
    f = ops.sample_rows(v)
    x.normal_()
    f(x, u, out=out, **p)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        f(x, u, out=out, **p)
    for i in range(5):
        x.copy_(torch.from_numpy(rng.standard_normal((rows, v)).astype(np.float32) * np.float32(2.0)))
        u.copy_(torch.from_numpy(rng.random(rows)))
        for k, t in params(rng, rows).items():
            p[k].copy_(t)
        g.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, f(x, u, **p))


def test_two_streams(ops, hip_device):
    rng = np.random.default_rng(15)
    sets = [(torch.from_numpy(rng.standard_normal((r, 60000)).astype(np.float32)).to(hip_device),
             torch.from_numpy(rng.random(r)).to(hip_device)) for r in (5, 30)]
    f = ops.sample_rows(60000)
    want = [f(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(f(*sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[i]) for i in range(2) for t in got[i])


def test_python_refusals(ops, hip_device):
    x = torch.zeros(4, 100, device=hip_device)
    u = torch.zeros(4, device=hip_device, dtype=torch.float64)
    f = ops.sample_rows(100)
    bits = torch.zeros(4, 4, device=hip_device, dtype=torch.int32)
    for args, kw in [((x[:, :99], u), {}), ((x.double(), u), {}), ((x.half(), u), {}), ((x.cpu(), u), {}), ((x[0], u), {}),
                     ((x.t().contiguous().t(), u), {}), ((x[:1].expand(4, 100), u), {}), ((x, u.float()), {}), ((x, u[:3]), {}),
                     ((x, u.cpu()), {}), ((x, u), dict(temperature=u)), ((x, u), dict(top_k=u.long())), ((x, u), dict(top_p=u)),
                     ((x, u), dict(min_p=u.float()[:3])), ((x, u), dict(cfg_scale=u.float())), ((x, u), dict(allowed=bits[:, :3])),
                     ((x, u), dict(allowed=bits[:3])), ((x, u), dict(allowed=bits.long())), ((x, u), dict(out=bits[:, 0])),
                     ((x, u), dict(logprob=u)), ((x, u), dict(kept=u.float()))]:
        with pytest.raises(ValueError):
            f(*args, **kw)
    g = ops.sample_rows(100, cfg=True)
    with pytest.raises(ValueError, match="cfg_scale"):
        g(x.view(2, 2, 100), u[:2])
    with pytest.raises(ValueError):
        g(x, u, cfg_scale=u.float())


@pytest.mark.parametrize("rows", [1, 3])
def test_a_slice_past_4096_below_a_largest_within(ops, hip_device, rows):
    """Largest values within 4,096 of 0 in one workgroup's part of the row, those of the other parts just past it."""
    rng = np.random.default_rng(44)
    V = 20000
    x = -4101 - 6 * rng.random((rows, V))
    x[:, 15000] = -4094.5
    x[:, 15003] = -4095
    x[-1, 9] = -4096.5
    p = dict(top_p=torch.full((rows,), 0.97), top_k=torch.tensor([0, 5000, 0][:rows], dtype=torch.int32))
    for u in (0.01, 0.3, 0.6, 0.95):
        check(ops, hip_device, torch.from_numpy(x.astype(np.float32)), [u] * rows, least=1.0, **p)


@pytest.mark.parametrize("fall", [3.0, 14.0, 40.0])
def test_parts_of_a_row_far_apart(ops, hip_device, fall):
    """Each part's largest value a good deal below the one before, bounds far below the row's largest: sums of parts are
    counted from refs of their own."""
    rng = np.random.default_rng(45)
    V, rows = 40000, 8
    x = 2.0 * rng.standard_normal((rows, V)) - np.linspace(0, fall, V)
    x[1::2] = x[1::2, ::-1]
    p = dict(top_k=torch.tensor([0, 20000, 35000, 3000, 0, 0, 39000, 12000], dtype=torch.int32),
             min_p=torch.tensor([1e-12, 0, 0, 1e-8, 1e-5, 1e-3, 0, 1e-10]), top_p=torch.tensor([1, 0.999999, 1, 1, 1, 0.9999, 0.99, 1.0]))
    for u in (0.2, 0.999):
        check(ops, hip_device, torch.from_numpy(x.astype(np.float32)), [u] * rows, least=0.8, **p)


@pytest.mark.parametrize("v", [100, 2051, 40000])
def test_the_only_one_has_logarithm_0(ops, hip_device, v):
    rng = np.random.default_rng(46)
    x = 3 * torch.from_numpy(rng.standard_normal((6, v)).astype(np.float32))
    p = dict(temperature=torch.tensor([0.7, 1.0, 1.3, 0.9, 1.0, 0.0]), top_k=torch.tensor([1, 1, 0, 0, 2000, 0], dtype=torch.int32),
             top_p=torch.tensor([0, 0.5, 1e-9, 0, 1e-6, 0]), min_p=torch.tensor([0, 0, 0, 1.0, 0, 0]))
    got, logprob, kept = sample(ops, hip_device, x, [0.7] * 6, **p)
    assert (got == x.argmax(1).numpy()).all() and (kept == 1).all() and (logprob == 0).all()


@pytest.mark.parametrize("v", [4095, 4096, 4097, 7001, 12000])
def test_rows_around_what_threads_hold(ops, hip_device, v):
    """One workgroup, the row in its threads' registers or read again for each step, by pieces or value by value."""
    for dtype in (F32, BF16):
        test_sizes(ops, hip_device, v, dtype)
        test_guidance_and_allowed(ops, hip_device, v, dtype)
    test_equal_values(ops, hip_device, v)
    # of 12,000, two rows' two largest are equal and alone after top-k, with a top_p of 0.5: its bound 0.5 (w + w) is the first
    # sum w itself, which no rounding decides, so 14 of 16 rows are determined
    test_close_values(ops, hip_device, v, least=0.875)
    test_masked_and_infinite_values(ops, hip_device, v)
    test_temperatures(ops, hip_device, v, 1e-4)
    test_ends_of_the_draw(ops, hip_device, v)


@pytest.mark.parametrize("v", [16500, 16501])
def test_many_long_rows_are_whole(ops, hip_device, v):
    """So many rows that each is one workgroup's, longer than those of few are."""
    rng = np.random.default_rng(v)
    rows = 300
    for dtype in (F32, BF16):
        x = torch.from_numpy(rng.standard_normal((rows, 2, v)).astype(np.float32) * np.float32(2.0)).to(dtype)
        scale = torch.from_numpy(rng.uniform(0.0, 3.0, rows).astype(np.float32))
        p = params(rng, rows)
        check(ops, hip_device, x, rng.random(rows), cfg=True, allowed=rng.random((1, v)) < 0.7, cfg_scale=scale, **p)
        check(ops, hip_device, x[:, 0].contiguous(), rng.random(rows), **p)
