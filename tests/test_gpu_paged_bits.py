"""The paged operators on inputs where low bits decide (paged_bits.py)."""

import numpy as np
import pytest
import torch

import paged_bits as bits
import paged_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TYPES = {"f32": (F32, F32), "f32_on_bf16": (F32, BF16), "bf16": (BF16, BF16)}
# few rows, and chunks that reach the kernels of 32 and 128 rows
SHAPES = {"few": ([(9, 20), (3, 40), (1, 2)], (4, 2)), "tiles": ([(150, 150), (40, 70)], (64, 64)),
          "rows32": ([(20, 90), (17, 60), (31, 31), (2, 40)], (64, 64))}


@pytest.fixture(scope="module")
def ops(hip_device):
    from soraku_amd import ops as O

    return O


def attend(ops, dev, u, scale, window):
    d = u.on(dev)
    lse = torch.empty(u.T, u.Hq, device=dev)
    out = ops.paged_attention(u.Hq, u.Hkv, u.hd, 16, scale, window)(d["q"], d["k"], d["v"], d["table"], d["starts"],
                                                                    d["lens"], lse=lse)
    return out.double().cpu().numpy(), lse.cpu().numpy()


def check(got, want, bound):
    off = np.abs(got - want)
    bad = np.argwhere(~(off <= bound))
    assert len(bad) == 0, (len(bad), bad[:5], float(off[tuple(bad.T)].max()))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("types", TYPES)
def test_weights(ops, hip_device, types, shape, hd):
    seqs, heads = SHAPES[shape]
    u, scale = bits.near_ties(seqs, heads, hd, *TYPES[types], seed=hd)
    check(attend(ops, hip_device, u, scale, 2)[0], *bits.out_bound(u, scale, 2))


@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("shape", [*SHAPES, "cuts"])
@pytest.mark.parametrize("types", TYPES)
def test_large_scores(ops, hip_device, types, shape, hd):
    """Scores around 1,024: the differences decide, in every wave and cut and across them."""
    seqs, heads = dict(SHAPES, cuts=([(1, 700), (1, 430)], (4, 2)))[shape]
    u, scale = bits.near_ties(seqs, heads, hd, *TYPES[types], seed=hd, level=128)
    check(attend(ops, hip_device, u, scale, 0)[0], *bits.out_bound(u, scale, 0))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES)
def test_queries(ops, hip_device, shape, hd):
    seqs, heads = SHAPES[shape]
    u, scale = bits.low_queries(seqs, heads, hd, seed=hd)
    check(attend(ops, hip_device, u, scale, 2)[0], *bits.out_bound(u, scale, 2))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("seqs", [[(20, 20), (3, 40)], [(1, 33), (1, 60)]])
def test_accounts_of_low_queries(ops, hip_device, seqs, hd):
    u, scale = bits.low_queries(seqs, (4, 2), hd, seed=hd)
    u.mass.zero_()
    d = u.on(hip_device)
    lse = torch.from_numpy(ref.attention(u, scale)[1].astype(np.float32))
    got = ops.paged_attention_mass(4, 2, hd, 16, scale)(d["q"], lse.to(hip_device), d["k"], d["table"], d["starts"],
                                                        d["lens"], d["mass"])
    check(got.double().cpu().numpy(), *bits.mass_bound(u, scale, lse.numpy()))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("swap", [False, True])
def test_accounts_of_low_products(ops, hip_device, swap, hd):
    """Chunks over FP32 caches: the products of low parts of both sides count."""
    u, scale = bits.low_products([(40, 40), (23, 90)], (4, 2), hd, swap, seed=hd)
    d = u.on(hip_device)
    lse = torch.from_numpy(ref.attention(u, scale)[1].astype(np.float32))
    got = ops.paged_attention_mass(4, 2, hd, 16, scale)(d["q"], lse.to(hip_device), d["k"], d["table"], d["starts"],
                                                        d["lens"], d["mass"])
    check(got.double().cpu().numpy(), *bits.mass_bound(u, scale, lse.numpy()))
