"""Projections with 8-bit weights on the GPU, each against its formula in 64 bits
(int8_ref.py): codes at ties and extremes, products of every kernel's sizes and of odd ones, norms,
SwiGLU, residuals in place, rows that hold infinities, graphs and streams."""

import numpy as np
import pytest
import torch

import int8_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops(hip_device):
    from soraku_amd import ops as O

    return O


def f32(t):
    return t.float().cpu().numpy()


def check_codes(ops, x, dev):
    got, scale = ops.int8_rows(x.shape[1])(x.to(dev))
    want, ws = ref.codes(f32(x))
    got, scale = got.cpu().numpy(), scale.cpu().numpy()
    assert got.shape == want.shape
    bad = np.argwhere(got != want)
    assert not len(bad), (bad[:5], got[tuple(bad[0])], want[tuple(bad[0])])
    assert np.array_equal(scale.view(np.int32)[~np.isnan(ws)], ws.view(np.int32)[~np.isnan(ws)])
    assert np.isnan(scale[np.isnan(ws)]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 3, 1025])
@pytest.mark.parametrize("k", [1, 7, 8, 100, 128, 130, 512, 1000, 1024, 1537, 2048, 2049, 4096, 4104, 8192, 8193, 20000])
def test_codes(ops, hip_device, rows, k, dtype):
    if rows * k > 3e6:
        rows = 130
    g = torch.Generator().manual_seed(rows * 7 + k)
    check_codes(ops, (torch.randn(rows, k, generator=g) * torch.randn(rows, 1, generator=g).exp()).to(dtype), hip_device)


def test_codes_of_the_longest_row(ops, hip_device):
    g = torch.Generator().manual_seed(2)
    check_codes(ops, torch.randn(2, 130944, generator=g), hip_device)
    check_codes(ops, torch.randn(3, 130943, generator=g).to(BF16), hip_device)


@pytest.mark.parametrize("k", [256, 300, 9000])
def test_codes_at_ties(ops, hip_device, k):
    """Middles between two codes and their neighbours, for tops with which 127 x / top is a middle exactly (127 times
    a power of two) and tops with which it never is."""
    r = np.random.default_rng(k)
    rows = []
    for top in [127.0, 127 * 2.0 ** -20, 127 * 2.0 ** 100, 63.5, 1.0, 3.0, 0.7, 1.9999999, 2.0 ** -130, 127 * 2.0 ** -149, 3.1e38]:
        top = np.float32(top)
        half = (r.integers(-127, 127, k) + 0.5).astype(np.float64)
        x = (half * np.float64(top) / 127).astype(np.float32)
        step = r.integers(-2, 3, k)
        for _ in range(2):
            x = np.where(step > 0, np.nextafter(x, np.float32(np.inf)), np.where(step < 0, np.nextafter(x, np.float32(-np.inf)), x))
            step = step - np.sign(step)
        x = np.clip(x, -top, top).astype(np.float32)
        x[r.integers(k)] = top
        rows.append(x)
    check_codes(ops, torch.from_numpy(np.stack(rows)), hip_device)
    check_codes(ops, torch.from_numpy(np.stack(rows)).to(BF16), hip_device)


@pytest.mark.parametrize("k", [5, 640, 8200])
def test_codes_of_rows_without_any(ops, hip_device, k):
    """Zeros, negative zeros, denormals, one value, the largest numbers, infinities and NaN."""
    x = torch.zeros(12, k)
    x[1] = -0.0
    x[2, 0] = 2.0 ** -149
    x[3] = torch.arange(k) * 2.0 ** -149
    x[4, k - 1] = -3.4e38
    x[5] = 3.4028234e38
    x[6, 1], x[6, 2] = float("inf"), 1.0
    x[7, k - 1] = float("nan")
    x[8, 0], x[8, k - 1] = -float("inf"), float("nan")
    x[9] = -1.0
    x[10, :3] = torch.tensor([2.0 ** -61, 2.0 ** -60, -(2.0 ** -62)])
    x[11, :3] = torch.tensor([2.0 ** -126, 2.0 ** -127, -(2.0 ** -126)])
    check_codes(ops, x, hip_device)
    check_codes(ops, x.to(BF16), hip_device)


def make(m, n, k, dtype, *, norm=False, swiglu=False, bias=False, residual=False, seed=0):
    g = torch.Generator().manual_seed(seed * 1009 + m * 31 + n * 7 + k)
    both = 2 * n if swiglu else n
    x = torch.randn(m, k, generator=g) * torch.randn(m, 1, generator=g).exp()
    w, ws = ref.codes((torch.randn(both, k, generator=g) * k ** -0.5).numpy())
    return dict(x=x.to(dtype), codes=torch.from_numpy(w), scales=torch.from_numpy(ws),
                gain=torch.randn(k, generator=g) * 0.2 + 1 if norm else None,
                bias=torch.randn(both, generator=g) if bias else None,
                residual=torch.randn(m, n, generator=g).to(dtype) if residual else None)


def on(d, dev):
    return {k: None if v is None else v.to(dev) for k, v in d.items()}


def expected(d, eps, swiglu):
    np_ = {k: None if v is None else (v.numpy() if k in ("codes", "scales") else f32(v)) for k, v in d.items()}
    return ref.linear(np_["x"], np_["codes"], np_["scales"], np_["gain"], eps, np_["bias"], np_["residual"], swiglu, d["x"].dtype == BF16)


def check_linear(ops, m, n, k, dtype, dev, eps=None, swiglu=False, **kw):
    d = make(m, n, k, dtype, swiglu=swiglu, **kw)
    got = ops.int8_linear(n, k, act="swiglu" if swiglu else None, eps=eps)(**on(d, dev))
    assert got.dtype == dtype and got.shape == (m, n)
    want, off = expected(d, eps, swiglu)
    half = ref.HALF_STEP[str(dtype)[6:]]
    err = np.abs(got.double().cpu().numpy() - want)
    lim = off + (np.abs(want) + off) * half + 2.0 ** -133
    assert (err <= lim).all(), (np.argwhere(~(err <= lim))[:5], np.nanmax(err / lim))


OPTIONS = {"plain": {}, "norm": dict(norm=True, eps=1e-6), "bias": dict(bias=True), "residual": dict(residual=True),
           "swiglu": dict(swiglu=True), "all": dict(norm=True, eps=1e-5, swiglu=True, bias=True, residual=True),
           "bare_norm": dict(eps=1e-6, residual=True)}
ROWS = [1, 2, 3, 5, 8, 9, 16, 17, 32, 33, 64, 65, 100, 129, 257, 400]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("options", OPTIONS)
@pytest.mark.parametrize("m", ROWS)
def test_linear_rows(ops, hip_device, m, options, dtype):
    for n, k in ((48, 256), (51, 300)):
        check_linear(ops, m, n, k, dtype, hip_device, **OPTIONS[options])


@pytest.mark.parametrize("options", ["plain", "all"])
@pytest.mark.parametrize("n,k", [(1, 1), (1, 128), (7, 5), (16, 127), (17, 129), (130, 1000), (2051, 1024), (4096, 2048), (520, 6144),
                                 (33, 8200), (128, 20001)])
@pytest.mark.parametrize("m", [1, 4, 7, 20, 50, 70, 300])
def test_linear_sizes(ops, hip_device, m, n, k, options):
    check_linear(ops, m, n, k, F32 if (n + m) % 2 else BF16, hip_device, **OPTIONS[options])


@pytest.mark.parametrize("m,n,k,dtype", [(1000, 1030, 384, F32), (2100, 2048, 640, BF16), (777, 4096, 1024, F32)])
@pytest.mark.parametrize("options", ["norm", "all"])
def test_linear_of_many_rows(ops, hip_device, m, n, k, dtype, options):
    check_linear(ops, m, n, k, dtype, hip_device, **OPTIONS[options])


def test_any_byte_is_a_code(ops, hip_device):
    """Codes of -128, and bytes behind K that meet zeros; the largest sum that K allows."""
    for m in (2, 20, 90):
        d = make(m, 40, 130, F32)
        d["codes"] = torch.randint(-128, 128, (40, 256), dtype=torch.int8)
        got = ops.int8_linear(40, 130)(**on(d, hip_device))
        want, off = expected(d, None, False)
        assert (np.abs(got.double().cpu().numpy() - want) <= off + np.abs(want) * 2.0 ** -24).all()
        k = 130944
        one = ops.int8_linear(3, k)(torch.ones(m, k, device=hip_device), torch.full((3, k), -128, dtype=torch.int8, device=hip_device),
                                    torch.ones(3, device=hip_device))
        want = -128.0 * k
        assert (np.abs(one.double().cpu().numpy() - want) <= 3 * 2.0 ** -24 * abs(want)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("eps", [None, 1e-6])
def test_a_row_does_not_hang_on_its_call(ops, hip_device, dtype, eps):
    """The same row alone, in a few and among many: the same bits, with the norm's sum too."""
    for n, k, swiglu in ((96, 1024, False), (77, 2100, True), (64, 9001, False)):
        d = on(make(700, n, k, dtype, norm=eps is not None, swiglu=swiglu, residual=True), hip_device)
        f = ops.int8_linear(n, k, act="swiglu" if swiglu else None, eps=eps)
        whole = f(**d)
        for m in (1, 2, 4, 7, 8, 12, 16, 30, 33, 64, 65, 120, 300):
            part = f(**dict(d, x=d["x"][:m], residual=d["residual"][:m]))
            assert torch.equal(part.view(torch.uint8), whole[:m].view(torch.uint8)), (n, k, m)
        big = dict(d, x=d["x"].repeat(3, 1), residual=d["residual"].repeat(3, 1))
        assert torch.equal(f(**big)[700:1400].view(torch.uint8), whole.view(torch.uint8))


@pytest.mark.parametrize("m", [2, 12, 40, 150])
def test_rows_with_infinities(ops, hip_device, m):
    """A row that holds an infinity or NaN gives NaN, alone; a row of zeros gives the bias."""
    d = on(make(m, 50, 200, F32, norm=True, bias=True), hip_device)
    f = ops.int8_linear(50, 200, eps=1e-6)
    clean = f(**d)
    x = d["x"].clone()
    x[m - 1, 7] = float("inf")
    x[0, 199] = float("nan")
    got = f(**dict(d, x=x))
    assert got[0].isnan().all() and got[m - 1].isnan().all()
    assert torch.equal(got[1: m - 1], clean[1: m - 1])
    x[0] = 0.0
    assert torch.equal(f(**dict(d, x=x))[0], d["bias"])


@pytest.mark.parametrize("m", [1, 6, 30, 64, 200])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_residual_in_place(ops, hip_device, m, dtype):
    for n in (64, 37):
        d = on(make(m, n, 512, dtype, residual=True), hip_device)
        f = ops.int8_linear(n, 512)
        want = f(**d)
        out = d["residual"].clone()
        assert f(**dict(d, residual=out), out=out) is out and torch.equal(out, want)


def test_no_rows(ops, hip_device):
    d = on(make(0, 16, 64, BF16), hip_device)
    assert ops.int8_linear(16, 64)(**d).shape == (0, 16)
    codes, scales = ops.int8_rows(64)(d["x"])
    assert codes.shape == (0, 128) and scales.shape == (0,)


def test_outputs_past_32_bits(ops, hip_device):
    """More than 2^32 bytes and 2^31 elements of output, codes past 2^31 bytes."""
    m, n, k = 1_050_000, 2056, 128
    g = torch.Generator(device=hip_device).manual_seed(3)
    x = torch.randn(m, k, generator=g, device=hip_device, dtype=BF16)
    codes = torch.randint(-127, 128, (n, k), generator=g, device=hip_device, dtype=torch.int8)
    scales = torch.rand(n, generator=g, device=hip_device)
    f = ops.int8_linear(n, k)
    out = f(x, codes, scales)
    for rows in (slice(0, 100), slice(m // 2, m // 2 + 77), slice(m - 133, m)):
        assert torch.equal(out[rows], f(x[rows].contiguous(), codes, scales))
    del out, x
    # codes of the activations themselves past 2^31 bytes
    m, k = 300_000, 8192
    x = torch.randn(m, k, generator=g, device=hip_device, dtype=BF16)
    codes = torch.randint(-127, 128, (16, k), generator=g, device=hip_device, dtype=torch.int8)
    f = ops.int8_linear(16, k)
    out = f(x, codes, scales[:16])
    for rows in (slice(0, 100), slice(m - 133, m)):
        assert torch.equal(out[rows], f(x[rows].contiguous(), codes, scales[:16]))


@pytest.mark.parametrize("m", [2, 24, 60, 200])
def test_captured_and_replayed(ops, hip_device, m):
    d = on(make(m, 256, 1024, F32, norm=True, swiglu=True, residual=True), hip_device)
    f = ops.int8_linear(256, 1024, act="swiglu", eps=1e-6)
    out = torch.empty(m, 256, device=hip_device)
    f(**d, out=out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        f(**d, out=out)
    for i in range(4):
        d["x"].copy_(torch.randn(m, 1024, generator=torch.Generator().manual_seed(i)))
        g.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, f(**d))


def test_two_streams(ops, hip_device):
    """Calls that run at the same time have workspaces of their own."""
    sets = [on(make(m, 512, 2048, BF16, norm=True, seed=i), hip_device) for i, m in enumerate((48, 300))]
    f = ops.int8_linear(512, 2048, eps=1e-6)
    want = [f(**d) for d in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(f(**sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_python_refusals(ops, hip_device):
    d = on(make(4, 32, 256, F32, bias=True, residual=True), hip_device)
    f = ops.int8_linear(32, 256)
    for name, bad in [("x", d["x"][:, :255]), ("x", d["x"].t().contiguous().t()), ("x", d["x"].double()), ("x", d["x"].half()),
                      ("x", d["x"].cpu()), ("x", d["x"][0]), ("codes", d["codes"][:31]), ("codes", d["codes"].int()),
                      ("codes", d["codes"].cpu()), ("scales", d["scales"].double()), ("scales", d["scales"][:31]),
                      ("bias", d["bias"].bfloat16()), ("residual", d["residual"].bfloat16()), ("residual", d["residual"][:3]),
                      ("gain", d["x"][0, :255])]:
        with pytest.raises(ValueError):
            f(**dict(d, **{name: bad}))
    with pytest.raises(RuntimeError, match="gain needs eps"):
        f(**dict(d, gain=d["x"][0].contiguous()))
    with pytest.raises(RuntimeError, match="out must not be x"):
        sq = on(make(4, 256, 256, F32), hip_device)
        ops.int8_linear(256, 256)(**sq, out=sq["x"])
    with pytest.raises(ValueError):
        f(**d, out=torch.empty(4, 31, device=hip_device))
    with pytest.raises(RuntimeError, match="aligned"):
        f(**dict(d, x=torch.randn(4 * 256 + 1, device=hip_device)[1:].view(4, 256)))
    with pytest.raises(ValueError):
        ops.int8_rows(256)(d["x"].double())
