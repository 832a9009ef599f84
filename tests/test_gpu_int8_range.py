"""8-bit projections of rows of any finite size: norms whose squares leave FP32's range, scales that sums of codes
would carry past it."""

import numpy as np
import pytest
import torch

import int8_ref as ref
from test_gpu_int8 import BF16, F32, expected, make, on

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(hip_device):
    from soraku_amd import ops as O

    return O


def check(ops, dev, d, n, k, eps, swiglu=False):
    got = ops.int8_linear(n, k, act="swiglu" if swiglu else None, eps=eps)(**on(d, dev)).double().cpu().numpy()
    want, off = expected(d, eps, swiglu)
    assert np.isfinite(want).all()
    lim = off + (np.abs(want) + off) * ref.HALF_STEP[str(d["x"].dtype)[6:]] + 2.0 ** -133
    assert (np.abs(got - want) <= lim).all(), (got[:, 0], want[:, 0])


# rows of one, a few, some and many, as the kernels divide them; K in registers, read twice, and not of whole pieces
SHAPES = [(1, 200), (2, 2048), (7, 1001), (7, 2048), (20, 512), (20, 1537), (90, 6144), (5, 8200), (40, 9001), (1100, 384), (1100, 2048)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("gain", [True, False])
@pytest.mark.parametrize("m,k", SHAPES)
def test_norms_of_any_finite_row(ops, hip_device, m, k, gain, dtype):
    n = 24
    d = make(m, n, k, dtype, norm=gain, bias=True, residual=True, seed=3)
    base = (d["x"].float() / d["x"].float().abs().amax(1, keepdim=True)).to(dtype)
    sizes = [1e20, 1.0, 1e30, 1e38, 1e19, 6e18, 1e-3]
    for eps, factors in ((1e-6, sizes), (0.0, sizes + [1e-15, 1e-19, 1e-25, 1e-34]), (1e-30, [1e-15, 1e-17, 1e-25, 1e22])):
        x = base.double()
        for r in range(m):
            x[r] *= factors[r % len(factors)] if m > 1 else factors[0]
        d["x"] = x.to(dtype)
        check(ops, hip_device, d, n, k, eps)
    if m == 1:
        for size in sizes[2:] + [1e-25]:
            d["x"] = (base.double() * size).to(dtype)
            check(ops, hip_device, d, n, k, 0.0)
    # one value whose square alone is past the range
    x = base.double()
    x[:, k - 1] = -3e25
    d["x"] = x.to(dtype)
    check(ops, hip_device, d, n, k, 1e-6)


@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_norms_do_not_hang_on_their_call(ops, hip_device, eps):
    for k in (1024, 1537):
        d = on(make(1200, 40, k, F32, norm=True, seed=4), hip_device)
        d["x"][::3] *= 1e22
        d["x"][1::3] *= 1e-22
        f = ops.int8_linear(40, k, eps=eps)
        whole = f(**d)
        for m in (1, 2, 5, 8, 9, 40, 300):
            assert torch.equal(f(**dict(d, x=d["x"][:m])), whole[:m])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,n,k", [(2, 40, 256), (7, 40, 300), (20, 40, 256), (70, 264, 384), (400, 264, 384), (3000, 264, 256)])
def test_sums_past_the_range_before_their_weights_scale(ops, hip_device, m, n, k, dtype):
    """Rows of up to 3e38 by weights of a usual size: outputs are finite, sums of codes times the row's scale alone are not."""
    d = make(m, n, k, dtype, bias=True, residual=True, seed=5)
    d["scales"] = d["scales"] * 2.0 ** -8
    top = d["x"].float().abs().amax(1, keepdim=True)
    size = torch.tensor([3e38, 1.0, 2e37, 1e30, 2.0 ** 103, 2.0 ** 104])[torch.arange(m) % 6][:, None]
    d["x"] = (d["x"].double() / top.double() * size.double()).to(dtype)
    check(ops, hip_device, d, n, k, None)


@pytest.mark.parametrize("m", [2, 20, 400])
def test_sums_of_zero_by_large_scales(ops, hip_device, m):
    """Sums that are 0 stay 0 where the two scales' product is past the range."""
    x = torch.full((m, 64), 3e38)
    x[:, 1::2] = -3e38
    codes = torch.zeros(70, 128, dtype=torch.int8)
    codes[:, :64] = 127
    bias = torch.arange(70.0)
    got = ops.int8_linear(70, 64)(x.to(hip_device), codes.to(hip_device), torch.full((70,), 1e15, device=hip_device), bias=bias.to(hip_device))
    assert torch.equal(got.cpu(), bias.expand(m, 70))
