"""Which kernels the 8-bit projections launch at the sizes that their GPU tests take for each tile
(stand-in HIP runtime)."""

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
