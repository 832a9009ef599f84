"""8-bit projections in each of their tiles against their formula in 64 bits (int8_ref.py): rows of the first tile, of the last two
and some between, every column."""

import numpy as np
import pytest
import torch

import int8_ref as ref
from int8_tiles import TILES
from test_gpu_int8 import BF16, F32, OPTIONS, f32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(hip_device):
    from soraku_amd import ops as O

    return O


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("options", ["plain", "all"])
@pytest.mark.parametrize("bm,bn,swiglu,m,n,k", TILES)
def test_tiles(ops, hip_device, bm, bn, swiglu, m, n, k, options, dtype):
    o = OPTIONS[options]
    g = torch.Generator().manual_seed(m + n + k)
    both = 2 * n if swiglu else n
    x = (torch.randn(m, k, generator=g) * torch.randn(m, 1, generator=g).exp()).to(dtype)
    codes = torch.randint(-127, 128, (both, k), generator=g).to(torch.int8)
    w = torch.nn.functional.pad(codes, (0, -k % 128))
    ws = (torch.rand(both, generator=g) + 0.5) * k ** -0.5 / 127
    gain = torch.randn(k, generator=g) * 0.2 + 1 if o.get("norm") else None
    bias = torch.randn(both, generator=g) if o.get("bias") else None
    res = torch.randn(m, n, generator=g).to(dtype) if o.get("residual") else None
    on = lambda t: None if t is None else t.to(hip_device)  # noqa: E731
    got = ops.int8_linear(n, k, act="swiglu" if swiglu else None, eps=o.get("eps"))(
        on(x), on(w), on(ws), gain=on(gain), bias=on(bias), residual=on(res))
    rows = torch.cat([torch.arange(bm), torch.arange(bm + 3, m - 2 * bm, 1 + m // 150), torch.arange(m - 2 * bm, m)])
    np_ = lambda t: None if t is None else f32(t)  # noqa: E731
    want, off = ref.linear(f32(x[rows]), w.numpy(), ws.numpy(), np_(gain), o.get("eps"), np_(bias),
                           None if res is None else f32(res[rows]), swiglu, dtype == BF16)
    err = np.abs(got[rows.to(hip_device)].double().cpu().numpy() - want)
    lim = off + (np.abs(want) + off) * ref.HALF_STEP[str(dtype)[6:]] + 2.0 ** -133
    if swiglu:
        # a gate below -126 ln 2 = -87.337 makes 1 + e^-g more than 2^126, whose reciprocal is denormal and counts as 0: silu is 0 in
        # place of g e^g, which falls in size from there on and is 87.34 * 2^-126 = 1.03e-36 there
        y, y_off = ref.linear(f32(x[rows]), w.numpy(), ws.numpy(), np_(gain), o.get("eps"), np_(bias))
        lim += np.where(y[:, :n] < -87.3, 1.03e-36 * 1.001 * (np.abs(y[:, n:]) + y_off[:, n:]), 0.0)
    assert (err <= lim).all(), (np.argwhere(~(err <= lim))[:5], np.nanmax(err / lim))
