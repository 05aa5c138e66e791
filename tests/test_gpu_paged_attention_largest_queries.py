"""Queries at the ends of their type, in prompts as in single tokens: the largest numbers, infinities
and NaN, value by value against the definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

from leanstack_amd import kernels

from paged_helpers import D
from test_gpu_paged_attention import check, ints, queries, setup

pytestmark = pytest.mark.gpu

MOST = 255 * 2.0 ** 120  # the largest bf16 number


@pytest.mark.parametrize("t", [1, 6, 70, 300])
@pytest.mark.parametrize("size", [MOST, 2.0 ** 127, 232 * 2.0 ** 120, 240 * 2.0 ** 120, 127 * 2.0 ** 120])
def test_largest_numbers(gpu, t, size):
    """|q| up to the type's largest over keys that leave the scores finite."""
    lens = [t + 60, t + 1]
    cache, table = setup(gpu, 2, 32, lens, seed=67)
    cache.exponents[0, 0] -= 40  # (of blocks that are not read, 255 is 215 then)
    q = queries(2, 8, t, seed=68).double()
    q = (q / q.abs().amax(-1, keepdim=True) * size).to(torch.bfloat16)
    assert float(q.abs().max()) == size
    got = check(gpu, cache, q, table, lens, 2.0 ** -88)
    assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("t", [5, 70])
def test_queries_that_are_not_finite_stay_apart(gpu, t):
    """An infinity or a NaN in some query rows: NaN there, the others as they are without."""
    lens = [t + 60, t + 1]
    cache, table = setup(gpu, 2, 32, lens, seed=69)
    q = queries(2, 8, t, seed=70)
    args = (cache, 0, ints(gpu, table), ints(gpu, lens), 0.1)
    want = kernels.paged_attention(q.to(gpu), *args).view(2, t, 8, D)
    bad = q.clone()
    bad[0, 3, 1, 17], bad[1, 0, t - 1, 100], bad[0, 7, 4, 0] = float("inf"), float("nan"), -float("inf")
    got = kernels.paged_attention(bad.to(gpu), *args).view(2, t, 8, D)
    nan = torch.zeros((2, t, 8), dtype=torch.bool)
    nan[0, 1, 3] = nan[1, t - 1, 0] = nan[0, 4, 7] = True
    assert torch.equal(torch.isnan(got).all(-1).cpu(), nan) and torch.equal(torch.isnan(got).any(-1).cpu(), nan)
    # (their waves may take another product: the same scores, added up in another order)
    off = (got.double() - want.double()).abs().cpu()[~nan]
    assert float(off.max()) <= 2.0 ** -8 * float(want.abs().max())


def test_padding_of_any_values(gpu):
    """Query tokens behind a request's count may hold anything."""
    lens, counts, t = [140, 70], [70, 33], 70
    cache, table = setup(gpu, 2, 32, lens, seed=71)
    q = queries(2, 8, t, seed=72)
    q[1, :, 33:] = float("nan")
    q[1, ::2, 40:] = MOST
    got = check(gpu, cache, q, table, lens, 0.1, counts)
    assert not got[1, 33:].any()
