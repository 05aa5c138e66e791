"""Queries whose dims are far apart, in prompts as in single tokens, value by value against the
definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

from paged_helpers import D, places
from test_gpu_paged_attention import check, queries, setup

pytestmark = pytest.mark.gpu


def without_dims(cache, dims):
    """The cache's keys with zeros in these dims."""
    for dim in dims:
        at = torch.from_numpy(places()[0][:, dim]).to(cache.storage.device)
        cache.storage[0, 0].index_fill_(-1, at, 0)


@pytest.mark.parametrize("t", [1, 5, 70, 200])
@pytest.mark.parametrize("power", [6, 10, 13, 16, 20, 24, 60, 120])
def test_one_large_dim_that_meets_zeros(gpu, t, power):
    """Scores are those of the other dims alone, however much smaller they are."""
    lens = [t + 100, t + 7]
    cache, table = setup(gpu, 2, 32, lens, seed=60)
    without_dims(cache, [5, 77])
    q = queries(2, 8, t, seed=61)
    q[:, :, ::3, 5] = 2.0 ** power
    q[:, 4:, 1::3, 77] = -2.0 ** power
    check(gpu, cache, q, table, lens, 0.1)


@pytest.mark.parametrize("t", [3, 70])
@pytest.mark.parametrize("dims", [1, 2, 5, 16, 64, 127])
def test_small_dims_beside_large_ones(gpu, t, dims):
    """`dims` dims 2^14..2^18 times smaller than the others, which the keys do not have."""
    lens = [150, 90]
    cache, table = setup(gpu, 2, 32, lens, seed=62)
    large = list(range(dims, D))
    without_dims(cache, large)
    q = queries(2, 8, t, seed=63).float()
    q[..., :dims] = q[..., :dims] * torch.exp2(-torch.arange(14, 19).float()[torch.arange(dims) % 5]) * 2.0 ** 10
    q[..., large] *= 2.0 ** 10
    check(gpu, cache, q.to(torch.bfloat16), table, lens, 20.0)


@pytest.mark.parametrize("t", [3, 70])
@pytest.mark.parametrize("low,high", [(-120, -100), (-126, -60), (-40, 40), (-133, -120), (-8, 8)])
def test_any_exponents(gpu, t, low, high):
    """Every value with an exponent of its own, subnormal numbers among them."""
    lens = [150, 90]
    cache, table = setup(gpu, 2, 32, lens, seed=64)
    gen = torch.Generator().manual_seed(65)
    q = queries(2, 8, t, seed=66).double() * torch.exp2(torch.randint(low, high + 1, (2, 8, t, D), generator=gen).double())
    scale = 2.0 ** -high if high < 120 else 1.0
    check(gpu, cache, q.to(torch.bfloat16), table, lens, min(scale, 2.0 ** 119))


@pytest.mark.parametrize("at", [0, 31, 32, 63, 64, 100, 127])
def test_a_wide_row_among_others(gpu, at):
    """One query row of a wave is wide; three small dims beside a large one, wherever they lie."""
    t = 70
    lens = [t + 300, t]
    cache, table = setup(gpu, 2, 32, lens, seed=73)
    q = queries(2, 8, t, seed=74)
    dims = [(at + i * 64 % 128 + i) % D for i in range(7)]
    without_dims(cache, [d for d in range(D) if d not in dims])
    q[1, 5, 40] = 2.0 ** 12
    q[1, 5, 40, dims] = (torch.arange(1, 8) * 2.0 ** -5).to(torch.bfloat16)
    q[0, 2, 69] = 2.0 ** 20
    q[0, 2, 69, dims] = (torch.arange(7, 0, -1) * 2.0 ** -3).to(torch.bfloat16)
    check(gpu, cache, q, table, lens, 1.0)
