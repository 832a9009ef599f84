"""The 8-bit projections without a GPU: what their entry points refuse (before any HIP call), what
they launch, and the oracle of their GPU tests against exact fractions."""

import ctypes as C
import json
import math
import os
import subprocess
import sys
from fractions import Fraction

import numpy as np
import pytest

import int8_ref as ref
from conftest import ROOT

P = 4096          # an aligned address that nothing reads


@pytest.fixture(scope="module")
def L():
    from soraku_amd import _lib

    return _lib.load()


ROWS = dict(stream=None, R=3, K=200, xd=0, x=P, codes=P, scales=P)
LINEAR = dict(stream=None, M=3, N=48, K=200, xd=0, act=0, eps=-1.0, x=P, gain=None, codes=P, scales=P, bias=None, res=None,
              out=2 * P, ws=None, ws_bytes=0)
BAD_ROWS = [("R", -1), ("R", 2 ** 24), ("K", 0), ("K", -8), ("K", 130945), ("xd", 2), ("xd", -1), ("x", None), ("codes", None),
            ("scales", None), ("x", P + 4), ("codes", P + 8)]
BAD_LINEAR = [("M", -1), ("M", 2 ** 24), ("N", 0), ("N", -1), ("N", 2 ** 20 + 1), ("K", 0), ("K", 130945), ("xd", 2), ("act", 2),
              ("act", -1), ("eps", math.nan), ("eps", math.inf), ("gain", P), ("x", None), ("codes", None), ("scales", None), ("out", None),
              ("x", P + 4), ("codes", P + 1), ("res", P + 8), ("out", P + 4), ("out", P), ("ws", P + 8), ("M", 20)]


@pytest.mark.parametrize("field,value", BAD_ROWS)
def test_rows_refusals(L, field, value):
    assert L.sk_op_int8_rows(*dict(ROWS, **{field: value}).values()) == -1
    assert L.sk_last_error().decode()


@pytest.mark.parametrize("field,value", BAD_LINEAR)
def test_linear_refusals(L, field, value):
    assert L.sk_op_int8_linear(*dict(LINEAR, **{field: value}).values()) == -1
    assert L.sk_last_error().decode()


def test_linear_asks_for_its_workspace(L):
    n = C.c_int64(-1)
    assert L.sk_op_int8_linear_workspace(100, 48, 200, 1, 1, C.byref(n)) == 0 and n.value >= 100 * 256 + 400
    args = dict(LINEAR, M=100, xd=1, act=1, ws=P, ws_bytes=n.value - 1)
    assert L.sk_op_int8_linear(*args.values()) == -1 and str(n.value) in L.sk_last_error().decode()
    assert L.sk_op_int8_linear_workspace(100, 48, 200, 1, 1, None) == -1
    assert L.sk_op_int8_linear_workspace(100, 0, 200, 1, 1, C.byref(n)) == -1
    assert L.sk_op_int8_linear_workspace(0, 48, 200, 1, 1, C.byref(n)) == 0 and n.value == 0


def test_linear_refuses_more_than_a_launch_holds(L):
    n = C.c_int64(-1)
    sizes = dict(M=2 ** 24 - 1, N=2 ** 20, K=128)
    assert L.sk_op_int8_linear_workspace(*sizes.values(), 0, 0, C.byref(n)) == 0
    assert L.sk_op_int8_linear(*dict(LINEAR, **sizes, ws=P, ws_bytes=n.value).values()) == -1
    assert "several calls" in L.sk_last_error().decode()


def test_python_refusals():
    import torch

    from soraku_amd import ops

    for big in (2 ** 31, 2 ** 32 + 64, -2 ** 32):
        with pytest.raises(ValueError, match="K must be a 32-bit integer"):
            ops.int8_rows(big)
        with pytest.raises(ValueError, match="N must be a 32-bit integer"):
            ops.int8_linear(big, 64)
    with pytest.raises(ValueError, match="act"):
        ops.int8_linear(16, 64, act="gelu")
    for eps in (-1.0, math.nan):
        with pytest.raises(ValueError, match="eps"):
            ops.int8_linear(16, 64, eps=eps)
    with pytest.raises(ValueError, match="HIP device"):
        ops.int8_rows(64)(torch.zeros(2, 64))
    with pytest.raises(ValueError, match="HIP device"):
        ops.int8_linear(16, 64)(torch.zeros(2, 64), torch.zeros(16, 128, dtype=torch.int8), torch.zeros(16))


# ------------------------------------------------------------------ launches (stand-in HIP runtime)

SCRIPT = '''
import json
import test_int8_cpu as t
out = []
for case in json.load(open(sys.argv[3])):
    args = dict(t.LINEAR, **case)
    n = C.c_int64()
    _lib.check(L.sk_op_int8_linear_workspace(args["M"], args["N"], args["K"], args["xd"], args["act"], C.byref(n)))
    args.update(ws=t.P if n.value else None, ws_bytes=n.value)
    calls()
    rc = L.sk_op_int8_linear(*args.values())
    cs = calls()
    stub.stub_fail(b"hipLaunchKernel", 0)
    failed = L.sk_op_int8_linear(*args.values())
    stub.stub_fail(b"", -1)
    calls()
    out.append([rc, [c[0] for c in cs], kernels(cs), n.value, failed])
print(json.dumps(out))
'''


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("stub")
    so = tmp / "stub.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    os.path.join(ROOT, "tests", "hip_host_stub.cpp"), "-o", str(so)], check=True)

    def run(cases):
        (tmp / "s.py").write_text(SCRIPT)
        (tmp / "c.json").write_text(json.dumps(cases))
        env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "tests"))
        r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "host_engine.py"), str(so), str(tmp / "s.py"),
                            str(tmp / "c.json")], capture_output=True, text=True, env=env)
        assert r.returncode == 0, r.stderr
        return json.loads(r.stdout.strip().splitlines()[-1])
    return run


def test_launches(launches):
    """Nothing but kernels is asked of the device, few of them, and a launch that fails is an error."""
    rng = np.random.default_rng(4)
    cases = [dict(M=int(m), N=int(n), K=int(k), xd=int(rng.integers(2)), act=int(rng.integers(2)))
             for m in (1, 2, 4, 8, 9, 16, 33, 64, 65, 200, 774, 5999, 2 ** 24 - 1) for n, k in
             ((1, 1), (48, 200), (2051, 1024), (4096, 2048), (2048, 6144), (128, 130944), (2 ** 20, 64))]
    for c, (rc, calls, kern, ws, failed) in zip(cases, launches(cases)):
        if rc == -1:                                  # more tiles than a grid holds: refused before any launch
            assert calls == [] and c["M"] * c["N"] > 2 ** 40
            continue
        assert rc == 0 and set(calls) == {"hipLaunchKernel"} and failed == -5
        assert len(kern) <= (1 if ws == 0 else 3)
        for _, grid in kern:
            assert all(0 < g <= (2 ** 31 - 1 if i == 0 else 65535) for i, g in enumerate(grid))
    (rc, calls, *_), = launches([dict(M=0)])
    assert rc == 0 and calls == []


# ------------------------------------------------------------------ the oracle

def test_codes_by_fractions():
    r = np.random.default_rng(0)
    for top in (127.0, 1.0, 3.0, 0.7, 254 * 2.0 ** -140, 3.4e38):
        x = (r.integers(-127, 127, 400) + 0.5) / 127 * top
        x = np.concatenate([x, r.standard_normal(100) * top / 4, [top]]).clip(-top, top).astype(np.float32)
        x = np.concatenate([x, np.nextafter(x, np.float32(0)), -x])
        q, s = ref.codes(x[None])
        m = Fraction(float(np.abs(x).max()))
        assert q[0, : len(x)].tolist() == [round(127 * Fraction(float(v)) / m) for v in x]   # halves to even
        assert q.shape[1] % 128 == 0 and not q[0, len(x):].any()
        assert s[0] == np.float32(float(m)) / np.float32(127)


def test_codes_of_rows_without_any():
    x = np.zeros((4, 5), np.float32)
    x[1, 2], x[2, 0], x[3, 4] = np.inf, np.nan, 2.0 ** -149
    q, s = ref.codes(x)
    assert not q[:3].any() and s[0] == 0 and np.isnan(s[1:3]).all() and q[3].tolist()[:5] == [0, 0, 0, 0, 127]
