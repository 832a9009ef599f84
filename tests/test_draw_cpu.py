"""Sampling by row without a GPU: what its entry points refuse (before any HIP call), what they launch, and the
oracle of its GPU tests against the decode path's."""

import ctypes as C
import json
import os
import subprocess
import sys

import numpy as np
import pytest

import draw_ref as ref
from conftest import ROOT

P = 4096          # an aligned address that nothing reads


@pytest.fixture(scope="module")
def L():
    from soraku_amd import _lib

    return _lib.load()


SAMPLE = dict(stream=None, R=3, V=100, dt=0, logits=P, stride=100, u=P, temperature=P, top_k=P, top_p=P, min_p=P, cfg=None, allowed=None,
              apart=0, token=P, logprob=None, kept=None, ws=None, ws_bytes=0)
BAD = [("R", -1), ("R", 65536), ("V", 0), ("V", -5), ("V", 2 ** 20 + 1), ("dt", 2), ("dt", -1), ("stride", 99), ("stride", -100),
       ("logits", None), ("u", None), ("token", None), ("ws", P + 8)]


@pytest.mark.parametrize("field,value", BAD)
def test_refusals(L, field, value):
    assert L.sk_op_sample_rows(*dict(SAMPLE, **{field: value}).values()) == -1
    assert L.sk_last_error().decode()


def test_masks_and_workspaces(L):
    for apart in (-4, 1, 3):
        assert L.sk_op_sample_rows(*dict(SAMPLE, allowed=P, apart=apart).values()) == -1
    n = C.c_int64(-1)
    assert L.sk_op_sample_rows_workspace(3, 100, 0, C.byref(n)) == 0 and n.value == 0
    assert L.sk_op_sample_rows_workspace(3, 151936, 0, C.byref(n)) == 0 and n.value > 0
    args = dict(SAMPLE, V=151936, stride=151936, ws=P, ws_bytes=n.value - 1)
    assert L.sk_op_sample_rows(*args.values()) == -1 and str(n.value) in L.sk_last_error().decode()
    assert L.sk_op_sample_rows_workspace(3, 100, 0, None) == -1 and L.sk_op_sample_rows_workspace(3, 0, 0, C.byref(n)) == -1


def test_python_refusals():
    import torch

    from soraku_amd import ops

    for big in (2 ** 31, 2 ** 32 + 64):
        with pytest.raises(ValueError, match="V must be a 32-bit integer"):
            ops.sample_rows(big)
    with pytest.raises(ValueError, match="HIP device"):
        ops.sample_rows(8)(torch.zeros(2, 8), torch.zeros(2, dtype=torch.float64))


SCRIPT = '''
import json
import test_draw_cpu as t
out = []
for case in json.load(open(sys.argv[3])):
    args = dict(t.SAMPLE, **case)
    args["stride"] = args["V"]
    n = C.c_int64()
    _lib.check(L.sk_op_sample_rows_workspace(args["R"], args["V"], args["dt"], C.byref(n)))
    args.update(ws=t.P if n.value else None, ws_bytes=n.value)
    calls()
    rc = L.sk_op_sample_rows(*args.values())
    cs = calls()
    stub.stub_fail(b"hipLaunchKernel", 0)
    failed = L.sk_op_sample_rows(*args.values())
    stub.stub_fail(b"", -1)
    calls()
    out.append([rc, [c[0] for c in cs], kernels(cs), n.value, failed])
print(json.dumps(out))
'''


def test_launches(tmp_path):
    """Nothing but kernels is asked of the device, at most two, and a launch that fails is an error."""
    so = tmp_path / "stub.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    os.path.join(ROOT, "tests", "hip_host_stub.cpp"), "-o", str(so)], check=True)
    cases = [dict(R=r, V=v, dt=d) for r in (0, 1, 64, 65535) for v in (1, 2051, 16384, 16385, 151936, 2 ** 20) for d in (0, 1)]
    (tmp_path / "s.py").write_text(SCRIPT)
    (tmp_path / "c.json").write_text(json.dumps(cases))
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "host_engine.py"), str(so), str(tmp_path / "s.py"),
                        str(tmp_path / "c.json")], capture_output=True, text=True,
                       env=dict(os.environ, PYTHONPATH=os.path.join(ROOT, "tests")))
    assert r.returncode == 0, r.stderr
    for c, (rc, calls, kern, ws, failed) in zip(cases, json.loads(r.stdout.strip().splitlines()[-1])):
        assert rc == 0
        if c["R"] == 0:
            assert calls == [] and failed == 0
            continue
        assert set(calls) == {"hipLaunchKernel"} and failed == -5 and len(kern) == (2 if ws else 1)
        for _, grid in kern:
            assert all(0 < g <= (2 ** 31 - 1 if i == 0 else 65535) for i, g in enumerate(grid))


# ------------------------------------------------------------------ the oracle

def test_oracle_agrees_with_the_decode_path_s():
    from oracle import sampler

    rng = np.random.default_rng(3)
    for i in range(200):
        v = int(rng.choice([5, 40, 300]))
        x = (rng.standard_normal(v) * 3).astype(np.float32)
        x[rng.random(v) < 0.1] = -np.inf
        if not np.isfinite(x).any():
            continue
        t, k, p, u = (float(rng.choice([0.0, 0.7, 1.0])), int(rng.choice([0, 1, 7, 50])), float(rng.choice([0.0, 0.5, 0.95])), rng.random())
        got = ref.row(x, u, temperature=t, top_k=k, top_p=p)
        if got[3] > 1e-12:
            assert got[0] == sampler.sample(x, temperature=t, top_k=k, top_p=p, u=u)
        if t > 0:
            probs = sampler.filtered_probs((x / np.float32(t)).astype(np.float32), k, p)
            assert got[2] == (probs > 0).sum() and abs(np.exp(got[1]) - probs[got[0]]) < 1e-12
    assert np.array_equal(ref.merge(np.stack([x, x[::-1]])[None], [1.5])[0],
                          sampler.cfg_merge(x, x[::-1], 1.5), equal_nan=True)


def test_oracle_min_p():
    x = np.log(np.array([0.5, 0.25, 0.125, 0.0625, 0.0625]) * 8).astype(np.float32)
    assert ref.row(x, 0.0, min_p=0.2)[2] == 3 and ref.row(x, 0.99, min_p=0.2)[0] == 2
    assert ref.row(x, 0.99, min_p=1.0)[:1] == (0,) and ref.row(x, 0.99, min_p=1.5)[2] == 5
