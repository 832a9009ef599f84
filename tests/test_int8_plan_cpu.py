"""Which kernels the 8-bit projections launch at the sizes that their GPU tests take for each tile, and how large a
product one call takes (stand-in HIP runtime)."""

import pytest

from int8_tiles import TILES
from test_int8_cpu import launches  # noqa: F401


def test_tiles(launches):  # noqa: F811
    cases = [dict(M=m, N=n, K=k, xd=xd, act=int(swiglu)) for _, _, swiglu, m, n, k in TILES for xd in (0, 1)]
    for i, (rc, _, kern, _, _) in enumerate(launches(cases)):
        bm, bn, swiglu, *_ = TILES[i // 2]
        assert rc == 0 and len(kern) == 2
        want = f"tiles_kernelI{'ft'[i % 2]}Lb{int(swiglu)}ELi{bm}ELi{bn}E"
        assert want in kern[1][0], (cases[i], kern[1][0])
    assert {(bm, bn) for bm, bn, *_ in TILES} == {(256, 256), (192, 256), (128, 128), (64, 128), (64, 64)}


@pytest.mark.parametrize("act", [0, 1])
def test_products_of_2_to_the_35_outputs_are_taken(launches, act):  # noqa: F811
    """A launch has less than 2^32 threads, of 16 outputs at least; such products have 2,048 columns at least, which tiles of up to
    256 make an eighth more."""
    cases = [dict(M=min(2 ** 35 // n, 2 ** 24 - 1), N=n, K=k, xd=xd, act=act)
             for n in (1, 65, 1000, 2049, 2051, 4097, 6144, 10001, 65537, 2 ** 18 + 1, 2 ** 20) for k in (1, 200, 2048, 130944) for xd in (0, 1)]
    assert max(c["M"] * c["N"] for c in cases) > 2 ** 35 - 2 ** 20
    for c, (rc, calls, *_) in zip(cases, launches(cases)):
        assert rc == 0 and set(calls) == {"hipLaunchKernel"}, c
