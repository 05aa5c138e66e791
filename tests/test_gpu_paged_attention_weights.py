"""Up to 16 query rows per kv head (single tokens) the softmax' weights keep 16 bits, so that the result is
within little more than its own rounding to bf16 of the definition in 64 bits; with more rows they are bf16."""

from __future__ import annotations

import pytest
import torch

from leanstack_amd import kernels

from paged_helpers import D, Pool, attention
from test_gpu_paged_attention import check as check_coarse
from test_gpu_paged_attention import ints, queries, setup

pytestmark = pytest.mark.gpu


def check(gpu, cache, q, table, lens, scale, counts=None):
    """The bound of paged_helpers.attention with the weights' roundings at 2^-16 instead of h = 2^-8: a weight
    is the sum of two bf16 numbers, the second rounded to 2^-8 of what the first leaves, 2^-8 of the weight.
    The exponential (two units of fp32's last place, 2^-23) and its argument's rounding (exponents of
    at most 2^6 here: 2^-24 * 2^6 * ln 2) add 2^-17; a part's sums and their joining at most 2^-14 of fp32's."""
    b, n_q, t, d = q.shape
    if t * n_q // cache.num_key_value_heads > 16:
        check_coarse(gpu, cache, q, table, lens, scale, counts)
        return
    got = kernels.paged_attention(q.to(gpu), cache, 0, ints(gpu, table), ints(gpu, lens), scale,
                                  counts=None if counts is None else ints(gpu, counts)).cpu().double().view(b, t, n_q, D)
    pool = Pool(cache.storage[0], cache.exponents[0])
    want, coarse = attention(pool, q, table, lens, scale, counts)
    h = 2.0 ** -8
    # sum p |v|, as the coarse bound has it: h |out| + 2 (h + off) most (1 + h) + 1e-30
    pool_abs = Pool(cache.storage[0], cache.exponents[0])
    pool_abs.bytes[1] &= 0x7F
    most, _ = attention(pool_abs, q, table, lens, scale, counts)
    off = torch.where(most > 0, (coarse - h * want.abs() - 1e-30) / (2 * most * (1 + h)) - h, 0).clamp(min=0)
    bound = h * want.abs() + 2 * (2.0 ** -16 + 2.0 ** -17 + 2.0 ** -17 + off) * most + 1e-30
    over = (got - want).abs() > bound
    assert not bool(over.any()), f"{int(over.sum())} of {over.numel()} values off, worst {float(((got - want).abs() / bound).max())}"


@pytest.mark.parametrize("n_q,n_kv,page_rows,t,lens,counts", [
    (32, 8, 64, 1, [2, 15, 33, 64, 100], None),       # one launch
    (8, 1, 16, 1, [500, 48], None),
    (40, 8, 64, 1, [200, 77], None),
    (32, 8, 64, 4, [30, 100, 5], [4, 3, 1]),          # 16 query rows
    (32, 8, 32, 5, [5, 6, 33, 500], None),            # 20
    (32, 8, 64, 8, [8, 60, 300], [8, 5, 8]),          # 32
    (48, 2, 64, 1, [90, 3], None),
])
@pytest.mark.parametrize("wide", [False, True])
def test_weights(gpu, n_q, n_kv, page_rows, t, lens, counts, wide):
    cache, table = setup(gpu, n_kv, page_rows, lens, seed=80 + t)
    if wide:  # (a table of more than 2048 rows: two launches)
        table = [row + [-1] * (2100 // page_rows) for row in table]
    check(gpu, cache, queries(len(lens), n_q, t, seed=81), table, lens, 0.05, counts)


@pytest.mark.parametrize("t,n_q,n_kv", [(1, 32, 8), (1, 4, 1), (4, 8, 2), (5, 8, 2)])
def test_long(gpu, t, n_q, n_kv):
    lens = [9000, 40, 3333]
    cache, table = setup(gpu, n_kv, 64, lens, seed=82)
    check(gpu, cache, queries(3, n_q, t, seed=83), table, lens, 0.05)


def test_nan_and_far_scores_as_before(gpu):
    """Weights that vanish and a maximum that rises from step to step."""
    lens = [700]
    cache, table = setup(gpu, 2, 32, lens, seed=84)
    q = queries(1, 8, 1, seed=85)
    check(gpu, cache, q, table, lens, 1.0)
    got = kernels.paged_attention(q.to(gpu), cache, 0, ints(gpu, table), ints(gpu, lens), 1e3)
    assert bool(torch.isfinite(got).all())
