"""The paged-cache operators without a GPU: what their entry points refuse
(before any HIP call), what they launch, and the 64-bit oracle of their GPU tests against
a second form."""

import ctypes as C
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import paged_ref as ref
from conftest import ROOT

P = 4096          # an aligned address that nothing reads


@pytest.fixture(scope="module")
def L():
    from soraku_amd import _lib

    return _lib.load()


APPEND = dict(stream=None, T=3, S=2, Hq=16, Hkv=8, hd=128, page=16, n_pages=9, width=4, stride=4, xd=0, kd=1, eps=1e-6,
              qkv=P, q_gain=P, k_gain=P, inv_freq=P, positions=P, starts=P, lens=P, table=P, k=P, v=P, mass=None, out=2 * P)
ATTEND = dict(stream=None, T=3, S=2, Hq=16, Hkv=8, hd=128, page=16, n_pages=9, width=4, stride=4, xd=0, kd=1, scale=0.1,
              window=0, sinks=0, q=P, k=P, v=P, table=P, starts=P, lens=P, out=2 * P, lse=None, ws=None, ws_bytes=0)
MASS = dict(stream=None, T=3, S=2, Hq=16, Hkv=8, hd=128, page=16, n_pages=9, width=4, stride=4, xd=0, kd=1, scale=0.1,
            window=0, sinks=0, q=P, lse=P, k=P, table=P, starts=P, lens=P, mass=P, ws=None, ws_bytes=0)
EVICT = dict(stream=None, S=2, Hkv=8, hd=128, page=16, n_pages=9, width=4, stride=4, kd=1, keep=32, sinks=4, recent=8,
             k=P, v=P, mass=P, table=P, lens=P, to=2 * P, to_stride=2, to_width=2, new_lens=2 * P, kept=P)
ENTRY = {"append": ("sk_op_paged_append", APPEND), "attention": ("sk_op_paged_attention", ATTEND),
         "mass": ("sk_op_paged_attention_mass", MASS), "evict": ("sk_op_paged_evict", EVICT)}

SIZES = [("S", 0), ("Hkv", 0), ("Hkv", -8), ("hd", 48), ("hd", 256), ("hd", 0), ("page", 0), ("page", 24), ("page", -16),
         ("n_pages", 0), ("width", 0), ("stride", 3), ("width", 2 ** 27), ("kd", 2)]
ROWS = [("T", -1), ("T", 2 ** 24), ("T", 2 ** 27), ("Hq", 12), ("Hq", 0), ("Hq", 8192), ("xd", 2), ("xd", 3)]
WINDOW = [("scale", 0.0), ("scale", -1.0), ("scale", math.inf), ("scale", 3e38), ("scale", math.nan), ("window", -1), ("sinks", -1)]
BAD = {
    "append": [*ROWS, ("eps", -1.0), ("eps", math.nan), ("q_gain", None), ("k_gain", None), ("qkv", P + 4), ("v", P + 8),
               ("out", P), ("out", P + 2), ("q_gain", P + 4)] + [(n, None) for n in ("qkv", "inv_freq", "positions", "starts", "lens",
                                                                         "table", "k", "v", "out")],
    "attention": [*ROWS, *WINDOW, ("q", P + 4), ("k", P + 2), ("out", P), ("out", P + 8), ("ws", P + 4)] + [
        (n, None) for n in ("q", "k", "v", "table", "starts", "lens", "out")],
    "mass": [*ROWS, *WINDOW, ("q", P + 4), ("k", P + 2), ("ws", P + 8)] + [(n, None) for n in ("q", "lse", "k", "table", "starts", "lens",
                                                                              "mass")],
    "evict": [("keep", 0), ("keep", -5), ("sinks", -1), ("recent", -1), ("sinks", 25), ("sinks", 2 ** 31 - 1), ("keep", 33),
              ("to_width", 0), ("to_stride", 1), ("to", P), ("new_lens", P), ("k", P + 4), ("v", P + 4)] + [
                  (n, None) for n in ("k", "v", "mass", "table", "lens", "to", "new_lens", "kept")],
}


@pytest.mark.parametrize("entry,field,value", [(e, *b) for e in BAD for b in SIZES + BAD[e]])
def test_refusals(L, entry, field, value):
    from soraku_amd._lib import SK_EINVAL

    name, good = ENTRY[entry]
    args = dict(good)
    assert field in args
    args[field] = value
    if field == "width":
        args["stride"] = value
    assert getattr(L, name)(*args.values()) == SK_EINVAL
    assert L.sk_last_error().decode()


@pytest.mark.parametrize("entry", ["append", "attention", "mass"])
def test_bf16_activations_need_a_bf16_cache(L, entry):
    name, good = ENTRY[entry]
    assert getattr(L, name)(*dict(good, xd=1, kd=0).values()) == -1
    assert "bfloat16" in L.sk_last_error().decode()


def test_attention_asks_for_its_workspace(L):
    from soraku_amd._lib import SK_EINVAL, SK_OK

    n = C.c_int64(-1)
    sizes = (2, 2, 16, 8, 128, 16, 4096, 0, 1, 0, 0)
    assert L.sk_op_paged_attention_workspace(*sizes, C.byref(n)) == SK_OK and n.value > 0
    args = dict(ATTEND, T=2, width=4096, stride=4096, ws=P, ws_bytes=n.value - 1)
    assert L.sk_op_paged_attention(*args.values()) == SK_EINVAL
    assert str(n.value) in L.sk_last_error().decode()
    assert L.sk_op_paged_attention_workspace(*sizes, None) == SK_EINVAL
    assert L.sk_op_paged_attention_workspace(2, 0, *sizes[2:], C.byref(n)) == SK_EINVAL


def test_mass_asks_for_its_workspace(L):
    from soraku_amd._lib import SK_EINVAL, SK_OK

    n = C.c_int64(-1)
    sizes = (2000, 1, 16, 8, 128, 16, 150, 0, 1)
    assert L.sk_op_paged_attention_mass_workspace(*sizes, C.byref(n)) == SK_OK and n.value > 0
    args = dict(MASS, T=2000, S=1, width=150, stride=150, ws=P, ws_bytes=n.value - 1)
    assert L.sk_op_paged_attention_mass(*args.values()) == SK_EINVAL
    assert str(n.value) in L.sk_last_error().decode()
    assert L.sk_op_paged_attention_mass_workspace(*sizes, None) == SK_EINVAL
    assert L.sk_op_paged_attention_mass_workspace(2, 0, *sizes[2:], C.byref(n)) == SK_EINVAL


def test_python_refusals():
    """Wrong devices, shapes and types raise before the library is called."""
    from soraku_amd import ops

    k = torch.zeros(4, 2, 16, 16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="HIP device"):
        ops.paged_attention(4, 2, 16, 16)(torch.zeros(1, 4, 16), k, k, i[:, None], i, i)
    with pytest.raises(ValueError, match="HIP device"):
        ops.paged_evict(2, 16, 16, 4)(k[0], k[0], k, i[:, None], i, i[:, None])
    i32, cpu = torch.int32, -1                       # a CPU tensor's device number
    for bad in (torch.zeros(2, 3), torch.zeros(3, 2).t(), torch.zeros(2, 3, dtype=torch.float64)[:, :2],
                torch.zeros(2, 3)[:, :2]):
        with pytest.raises(ValueError, match="must be a contiguous"):
            ops._need(bad, "x", torch.float32, cpu, (2, 2))
    with pytest.raises(ValueError, match="HIP device 0"):
        ops._need(torch.zeros(2, 2), "x", torch.float32, 0, (2, 2))
    for bad in (i, i[:, None].long(), torch.zeros(3, 2, dtype=i32), torch.zeros(3, 2, dtype=i32).t(),
                torch.zeros(1, 3, dtype=i32).expand(2, 3)):
        with pytest.raises(ValueError):
            ops._table(bad, "table", i32, cpu, 2)
    wide = torch.zeros(2, 7, dtype=i32)
    assert ops._table(wide[:, :3], "table", i32, cpu, 2)[1:] == (7, 3)
    assert ops._table(wide[:1, :3], "table", i32, cpu, 1)[1:] == (3, 3)
    with pytest.raises(ValueError, match="not supported"):
        ops._code(torch.zeros(1, dtype=torch.float16), {torch.float32: 0})


@pytest.mark.parametrize("big", [2 ** 31, 2 ** 32, 2 ** 32 + 64, -2 ** 32])
def test_python_refuses_sizes_past_32_bits(big):
    """A foreign call would take 2^32 for 0 (a window that lets every slot be seen) and 2^32 + 64 for 64."""
    from soraku_amd import ops

    makers = {ops.paged_append: dict(Hq=4, Hkv=2, hd=16, page=16, eps=1e-6),
              ops.paged_attention: dict(Hq=4, Hkv=2, hd=16, page=16, window=8, sinks=2),
              ops.paged_attention_mass: dict(Hq=4, Hkv=2, hd=16, page=16, window=8, sinks=2),
              ops.paged_evict: dict(Hkv=2, hd=16, page=16, keep=16, sinks=2, recent=3)}
    for make, good in makers.items():
        assert callable(make(**good)) and callable(make(**{k: v if k == "eps" else np.int64(v) for k, v in good.items()}))
        for name in good:
            if name != "eps":
                with pytest.raises(ValueError, match=f"{name} must be a 32-bit integer"):
                    make(**dict(good, **{name: big}))
    if big > 0:
        with pytest.raises(ValueError, match="2.31"):
            ops._table(torch.empty(1, big, dtype=torch.int32, device="meta"), "table", torch.int32, -1, 1)
        with pytest.raises(ValueError, match="tokens"):
            ops._code(torch.empty(big, 1, device="meta"), {torch.float32: 0})


# ------------------------------------------------------------------ launches (stand-in HIP runtime)

SCRIPT = '''
import json
import test_paged_cpu as t
cases = json.load(open(sys.argv[3]))
out = []
for entry, change in cases:
    name, good = t.ENTRY[entry]
    args = dict(good, **change)
    if entry == "attention":
        n = C.c_int64()
        _lib.check(L.sk_op_paged_attention_workspace(*[args[k] for k in ("T", "S", "Hq", "Hkv", "hd", "page", "width", "xd",
                                                                         "kd", "window", "sinks")], C.byref(n)))
        args.update(ws=t.P if n.value else None, ws_bytes=n.value)
    if entry == "mass":
        n = C.c_int64()
        _lib.check(L.sk_op_paged_attention_mass_workspace(*[args[k] for k in ("T", "S", "Hq", "Hkv", "hd", "page", "width", "xd",
                                                                              "kd")], C.byref(n)))
        args.update(ws=t.P if n.value else None, ws_bytes=n.value)
    calls()
    rc = getattr(L, name)(*args.values())
    cs = calls()
    out.append([rc, [c[0] for c in cs], kernels(cs), args.get("ws_bytes", 0)])
    stub.stub_fail(b"hipLaunchKernel", 0)
    out[-1].append(getattr(L, name)(*args.values()))
    stub.stub_fail(b"", -1)
    calls()
print(json.dumps(out))
'''


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("stub")
    so = tmp / "stub.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    os.path.join(ROOT, "tests", "hip_host_stub.cpp"), "-o", str(so)], check=True)

    def run(cases, script=SCRIPT):
        import json

        (tmp / "s.py").write_text(script)
        (tmp / "c.json").write_text(json.dumps(cases))
        env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "tests"))
        r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "host_engine.py"), str(so), str(tmp / "s.py"),
                            str(tmp / "c.json")], capture_output=True, text=True, env=env)
        assert r.returncode == 0, r.stderr
        return json.loads(r.stdout.strip().splitlines()[-1])
    return run


def test_launches(launches):
    """Nothing but kernels is asked of the device, a launch that fails is an
    error, and no tokens means no launch."""
    from soraku_amd._lib import SK_EHIP, SK_OK

    cases = [[e, c] for e in ENTRY for c in ({}, {"kd": 0}, {"hd": 16, "stride": 9})]
    cases += [["attention", {"T": 1, "S": 1, "width": 4096, "stride": 4096}], ["mass", {"T": 3000, "S": 1}]]
    for (entry, _), (rc, calls, kern, ws, failed) in zip(cases, launches(cases)):
        assert rc == SK_OK and set(calls) == {"hipLaunchKernel"} and failed == SK_EHIP
        assert len(kern) == (2 if entry == "evict" or ws else 1)
        for _, grid in kern:
            assert all(0 < g <= (2 ** 31 - 1 if i == 0 else 65535) for i, g in enumerate(grid))
    for entry in ("append", "attention", "mass"):
        (rc, calls, *_), = launches([[entry, {"T": 0}]])
        assert rc == SK_OK and calls == []


def test_attention_plans_cover_rows_and_keys(launches):
    """Every row tile has a workgroup whatever way T rows fall on S sequences,
    and the cuts reach the table's end."""
    rng = np.random.default_rng(1)
    cases = []
    for _ in range(60):
        hkv = int(rng.choice([1, 2, 3, 8]))
        cases.append(["attention", dict(T=int(rng.integers(1, 400)), S=int(rng.integers(1, 40)), Hkv=hkv,
                                        Hq=hkv * int(rng.integers(1, 9)), width=int(rng.integers(1, 300)), stride=300,
                                        page=16 * int(rng.integers(1, 20)), window=int(rng.choice([0, 1, 700])),
                                        sinks=int(rng.choice([0, 5])))])
    for (_, c), (rc, _, kern, ws, _) in zip(cases, launches(cases)):
        assert rc == 0
        (name, grid) = kern[0]
        R, G = rows_of(name), c["Hq"] // c["Hkv"]
        assert grid[0] == c["Hkv"]
        for _ in range(20):                          # rows of the sequences, some with none
            cuts = np.sort(rng.integers(0, c["T"] + 1, c["S"] - 1))
            n = np.diff(np.concatenate(([0], cuts, [c["T"]])))
            assert sum(-(-int(x) * G // R) for x in n) <= grid[1]
        assert ws == ((grid[2] * (128 + 2) + 1) * c["T"] * c["Hq"] * 4 if grid[2] > 1 else 0)


class AttendArgs(C.Structure):
    """The kernels' argument (AttendArgs of sk_paged.h, a Cache first)."""

    _fields_ = [(n, C.c_void_p) for n in ("k", "v", "table")] + [("stride", C.c_int64), ("width", C.c_int32)] + [
        (n, C.c_void_p) for n in ("starts", "lens")] + [(n, C.c_int32) for n in ("T", "S", "Hq", "Hkv", "G", "n_pages", "page")] + [
        ("page_mul", C.c_uint32), ("page_shift", C.c_int32)] + [(n, C.c_void_p) for n in ("q", "out", "lse")] + [
        ("scale2", C.c_float)] + [(n, C.c_int32) for n in ("window", "sinks", "cut", "last")] + [
        (n, C.c_void_p) for n in ("part", "ml", "count")]


ARGS = f"stub.stub_keep_args({C.sizeof(AttendArgs)})\n" + SCRIPT.replace("kernels(cs)", "[c[5:] + c[1:4] for c in cs]")


def longest_walk(c, R, n, length):
    """Key tiles that a tile of R rows of a sequence of n new tokens and that length goes through, at most."""
    G, p0, most = c["Hq"] // c["Hkv"], length - n, 0
    for f in range(0, n * G, R):
        lo_slot, hi_slot = p0 + f // G, p0 + (min(f + R, n * G) - 1) // G
        lo = (lo_slot - c["window"] + 1) // 16 if 0 < c["window"] <= lo_slot else 0
        most = max(most, 0 if hi_slot < 0 else hi_slot // 16 + 1 - lo + min(-(-c["sinks"] // 16), lo))
    return most


@pytest.mark.parametrize("hd,xd,kd", [(16, 0, 0), (16, 1, 1), (32, 0, 1), (64, 1, 1), (128, 0, 0), (128, 0, 1), (128, 1, 1)])
def test_attention_cuts_reach_the_longest_walk(launches, hd, xd, kd):
    """Cuts are whole steps of four tiles and together as long as any walk can be, and the
    last row tile of a launch is the one that its grid ends at."""
    rng = np.random.default_rng(hd + xd + 2 * kd)
    cases = []
    for i in range(60):
        hkv = int(rng.choice([1, 2, 8, 64]))
        S = int(rng.choice([1, 2, 7, 40]))
        cases.append(["attention", dict(T=S * int(rng.choice([1, 1, 5, 70, 600])), S=S, Hkv=hkv, Hq=hkv * int(rng.choice([1, 2, 8])), hd=hd, xd=xd,
                                        kd=kd, width=(w := int(rng.choice([1, 9, 60, 300]))), stride=w, page=16 * int(rng.integers(1, 9)),
                                        window=int(rng.choice([0, 1, 40, 700])), sinks=int(rng.choice([0, 5, 100])))])
    some_cut = False
    for (_, c), (rc, _, kern, _, _) in zip(cases, launches(cases, ARGS)):
        assert rc == 0
        name, raw, *grid = kern[0]
        a, R, cap = AttendArgs.from_buffer_copy(bytes.fromhex(raw)), rows_of(name), c["width"] * c["page"]
        assert (a.T, a.S, a.G, a.page, a.window, a.sinks, a.width) == (c["T"], c["S"], c["Hq"] // c["Hkv"], c["page"],
                                                                       c["window"], c["sinks"], c["width"])
        gx, gy, gz = (int(x) for x in grid)
        assert a.cut > 0 and a.cut % 4 == 0 and a.last == gy - 1
        some_cut |= gz > 1
        n = c["T"] // c["S"]
        for length in (cap, max(1, cap - 7), int(rng.integers(1, cap + 1)), min(cap, n)):
            assert longest_walk(c, R, n, length) <= gz * a.cut
            assert longest_walk(c, R, c["T"], length) <= gz * a.cut
    assert some_cut


@pytest.mark.parametrize("entry", ["append", "attention", "mass", "evict"])
def test_most_sequences(L, launches, entry):
    """65,535 sequences run, more are refused, by the workspace queries too."""
    from soraku_amd._lib import SK_EINVAL, SK_OK

    (rc, *_), = launches([[entry, {"S": 65535, **({} if entry == "evict" else {"T": 65535})}]])
    assert rc == SK_OK
    name, good = ENTRY[entry]
    for S in (65536, 2 ** 31 - 1):
        assert getattr(L, name)(*dict(good, S=S).values()) == SK_EINVAL
        assert "S in [1, 65535]" in L.sk_last_error().decode()
    n = C.c_int64()
    assert L.sk_op_paged_attention_workspace(3, 65536, 16, 8, 128, 16, 4, 0, 1, 0, 0, C.byref(n)) == SK_EINVAL
    assert L.sk_op_paged_attention_mass_workspace(3, 65536, 16, 8, 128, 16, 4, 0, 1, C.byref(n)) == SK_EINVAL


@pytest.mark.parametrize("change", [dict(T=2 ** 21 + 5, hd=16, kd=0), dict(T=2 ** 24 - 1, hd=16, kd=0), dict(T=2 ** 23 + 77, hd=32, xd=1),
                                    dict(T=2 ** 24 - 1, S=40, hd=64), dict(T=65535 * 32, hd=16, kd=0)])
def test_attention_of_millions_of_rows(launches, change):
    """Row tiles past what a grid takes go into further launches; none is left out."""
    (rc, calls, kern, ws, _), = launches([["attention", dict(dict(Hq=1, Hkv=1, S=1, width=10, stride=10, page=2 ** 20), **change)]])
    assert rc == 0 and ws == 0
    R = {rows_of(name) for name, _ in kern}
    assert len(R) == 1 and all(grid[0] == grid[2] == 1 and 0 < grid[1] <= 65535 for _, grid in kern)
    assert sum(grid[1] for _, grid in kern) * R.pop() >= change["T"]
    assert all(grid[1] == 65535 for _, grid in kern[:-1])


@pytest.mark.parametrize("hd,kd,keys", [(16, 1, 128), (128, 0, 128), (128, 1, 256)])
def test_most_slots_of_accounts(L, launches, hd, kd, keys):
    """The limit that the header gives: refused past it, by the workspace query as by the call."""
    from soraku_amd._lib import SK_EINVAL, SK_OK

    width = 65535 * keys // 16
    base = dict(hd=hd, kd=kd, width=width, stride=width)
    (rc, _, kern, _, _), = launches([["mass", base]])
    assert rc == SK_OK and kern[0][1][1] == 65535
    n = C.c_int64()
    assert L.sk_op_paged_attention_mass(*dict(MASS, **dict(base, width=width + 1, stride=width + 1)).values()) == SK_EINVAL
    assert str(65535 * keys) in L.sk_last_error().decode()
    assert L.sk_op_paged_attention_mass_workspace(3, 2, 16, 8, hd, 16, width + 1, 0, kd, C.byref(n)) == SK_EINVAL
    assert L.sk_op_paged_attention_mass_workspace(3, 2, 16, 8, hd, 16, width, 0, kd, C.byref(n)) == SK_OK


@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 5)])
def test_attention_kernels_of_many_heads(launches, window, sinks):
    """The GPU tests' shapes reach the kernels that they are there for."""
    import re

    types = {"f32": (0, 0), "f32_on_bf16": (0, 1), "bf16": (1, 1)}
    cases, want = [], []
    for seqs, heads, width, kernels in ref.MANY_HEADS:
        for t, (xd, kd) in types.items():
            cases.append(["attention", dict(T=sum(n for n, _ in seqs), S=len(seqs), Hq=heads, Hkv=heads, hd=64, page=16,
                                            width=width, stride=width, xd=xd, kd=kd, window=window, sinks=sinks)])
            want.append(kernels[t])
    for (name, nt), (rc, _, kern, _, _) in zip(want, launches(cases)):
        assert rc == 0 and f"attend_{name}_kernel" in kern[0][0]
        assert name == "tiles" or int(re.findall(r"Li(\d+)E", kern[0][0])[1]) == nt


def rows_of(kernel):
    """Rows of a workgroup, by the kernel's name and template arguments."""
    import re

    args = [int(x) for x in re.findall(r"Li(\d+)E", kernel)]
    assert "attend_" in kernel, kernel
    return 128 if "attend_tiles_kernel" in kernel else 16 * args[1]


# ------------------------------------------------------------------ the oracle

@pytest.mark.parametrize("window,sinks", [(0, 0), (3, 2), (20, 0)])
def test_oracle_attention_and_mass(window, sinks):
    u = ref.Setup([(3, 20), (0, 5), (6, 6), (2, 1)], 4, 2, 16, 16, seed=1)
    out, lse, _, _ = ref.attention(u, None, window, sinks)
    acc, _ = ref.mass(u, lse, None, window, sinks)
    grown = acc - u.mass.double().numpy()
    for s, (n, length) in enumerate(u.seqs):
        if n == 0:
            continue
        pool = lambda x: x[torch.from_numpy(u.table[s]).long()].double().transpose(0, 1).flatten(1, 2)[:, :length]  # noqa: E731
        k, v = (pool(x).repeat_interleave(u.G, 0) for x in (u.k, u.v))
        q = u.q[u.starts[s]: u.starts[s + 1]].double().transpose(0, 1)
        p, j = torch.arange(length - n, length)[:, None], torch.arange(length)
        see = (j <= p) & ((j > p - window) | (j < sinks) if window else True)
        x = (q @ k.transpose(1, 2) / 4.0).masked_fill(~see, -math.inf)
        w = torch.softmax(x, -1).nan_to_num(0.0)
        want = (w @ v).transpose(0, 1)
        assert torch.allclose(torch.from_numpy(out[u.starts[s]: u.starts[s + 1]]), want)
        got = torch.from_numpy(grown)[torch.from_numpy(u.table[s]).long()].transpose(0, 1).flatten(1, 2)[:, :length]
        assert torch.allclose(got, w.sum(1).view(u.Hkv, u.G, -1).sum(1), atol=1e-12)


def test_oracle_evict_and_append():
    u = ref.Setup([(1, 9), (1, 30)], 2, 1, 16, 16, seed=2)
    u.mass = torch.zeros_like(u.mass)
    u.mass[u.table[1, 0], 0, 5] = 2.0
    u.mass[u.table[1, 1], 0, 3] = float("nan")
    lens, kept = ref.evict(u, 10, 2, 3)
    assert lens.tolist() == [9, 10] and kept[0, 0].tolist() == [*range(9), -1]
    assert kept[1, 0].tolist() == [0, 1, 2, 3, 4, 5, 19, 27, 28, 29]
    q, k, v, mass = ref.append(u, None, None, np.ones(8, np.float32), np.array([0, 1]), 0.0)
    x = u.qkv.double().numpy().reshape(2, 4, 16)
    assert np.allclose(q[0], x[0, :2]) and np.allclose(k[u.table[0, 0], 0, 8], x[0, 2])
    z = (x[1, 0, :8] + 1j * x[1, 0, 8:]) * np.exp(1j)
    assert np.allclose(q[1, 0], np.concatenate((z.real, z.imag))) and np.allclose(v[u.table[1, 1], 0, 13], x[1, 3])
    assert mass[u.table[1, 1], 0, 13] == 0.0
