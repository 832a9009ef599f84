"""The bounds of paged_bits.py: the kernels' arithmetic stays within them, and a part of a
value that is left out does not."""

import numpy as np
import pytest
import torch

import paged_bits as bits
import paged_ref as ref

F32, BF16 = torch.float32, torch.bfloat16
SEQS, HEADS = [(20, 20), (3, 40)], (4, 2)


def worst(got, want, bound):
    return float(np.max(np.abs(got - want) / bound))


def test_parts_add_up():
    x = np.random.default_rng(0).standard_normal(1000).astype(np.float32)
    assert np.array_equal(sum(bits.cut(x, 3)), x.astype(np.float64))
    assert np.abs(sum(bits.cut(x, 2)) / x - 1).max() <= 2.0 ** -16
    assert np.abs(bits.cut(x, 1)[0] / x - 1).max() <= 2.0 ** -8


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("xd,kd,parts", [(F32, BF16, 3), (F32, F32, 3), (BF16, BF16, 2)])
def test_weights(hd, xd, kd, parts):
    u, scale = bits.near_ties(SEQS, HEADS, hd, xd, kd, seed=hd)
    want, bound = bits.out_bound(u, scale, 2)
    assert worst(bits.simulate(u, scale, 2, 3, parts), want, bound) < 1
    assert worst(bits.simulate(u, scale, 2, 3, parts - 1), want, bound) > 2


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_queries(hd):
    u, scale = bits.low_queries(SEQS, HEADS, hd, seed=hd)
    want, bound = bits.out_bound(u, scale, 2)
    assert worst(bits.simulate(u, scale, 2, 3, 3), want, bound) < 1
    assert worst(bits.simulate(u, scale, 2, 2, 3), want, bound) > 1000


@pytest.mark.parametrize("swap", [False, True])
def test_products_of_accounts(swap):
    u, scale = bits.low_products(SEQS, HEADS, 32, swap, seed=5)
    lse = ref.attention(u, scale)[1].astype(np.float32)
    want, bound = bits.mass_bound(u, scale, lse)
    hit = bound > 0

    def off(keep):
        return worst(bits.simulate_mass(u, scale, lse, keep)[hit], want[hit], bound[hit])

    assert off(lambda i, j: True) < 1
    assert off(lambda i, j: i + j < 3) > 1000
    assert off(lambda i, j: (i, j) != ((2, 1) if swap else (1, 2))) > 1000


def test_low_queries_of_accounts():
    u, scale = bits.low_queries(SEQS, HEADS, 64, seed=6)
    u.mass.zero_()
    lse = ref.attention(u, scale)[1].astype(np.float32)
    want, bound = bits.mass_bound(u, scale, lse)
    hit = bound > 0
    assert worst(bits.simulate_mass(u, scale, lse, lambda i, j: True)[hit], want[hit], bound[hit]) < 1
    assert worst(bits.simulate_mass(u, scale, lse, lambda i, j: i < 2)[hit], want[hit], bound[hit]) > 1000
