"""Scores are sums in 32 bits, whatever their products: a few large ones do not swallow the others, and
large ones that cancel leave the rest, in prompts as in single tokens."""

from __future__ import annotations

import pytest
import torch

from paged_helpers import D, places
from test_gpu_paged_attention import check, queries, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1, 5, 16, 70, 200])
@pytest.mark.parametrize("power", [2, 4, 6, 8, 10])
@pytest.mark.parametrize("scale", [1.0, 0.1])
def test_large_products_beside_small_ones(gpu, t, power, scale):
    """Some dims of every query are 2^power times the others."""
    lens = [t + 100, t + 7]
    cache, table = setup(gpu, 2, 32, lens, seed=90)
    q = queries(2, 8, t, seed=91)
    q[..., [9, 70, 127]] *= 2.0 ** power
    check(gpu, cache, q, table, lens, scale)


@pytest.mark.parametrize("t", [1, 5, 16, 70, 200])
@pytest.mark.parametrize("power", [4, 8, 12])
@pytest.mark.parametrize("pair", [(0, 1), (0, 7), (3, 8), (40, 41), (30, 33), (63, 64), (5, 100)])
def test_large_products_that_cancel(gpu, t, power, pair):
    """Two dims whose products are large and add up to zero for every key."""
    lens = [t + 100, t + 7]
    cache, table = setup(gpu, 2, 32, lens, seed=92)
    one, other = (torch.from_numpy(places()[0][:, dim]).to(cache.storage.device) for dim in pair)
    keys = cache.storage[0, 0]
    stale = (keys[..., one] & 0x7F) == 0x7F
    keys[..., other] = torch.where(stale, 0x7F, keys[..., one] ^ 0x80).to(torch.uint8)
    q = queries(2, 8, t, seed=93)
    q[..., pair[1]] = q[..., pair[0]] = q[..., pair[0]] * 2.0 ** power
    check(gpu, cache, q, table, lens, 1.0)


@pytest.mark.parametrize("t", [5, 70, 200])
@pytest.mark.parametrize("seed", range(6))
def test_keys_with_large_dims(gpu, t, seed):
    """Keys of which some dims are large in every row, as outlier channels are."""
    lens = [t + 150, t + 31]
    cache, table = setup(gpu, 2, 32, lens, seed=94 + seed)
    q = queries(2, 8, t, seed=100 + seed)
    gen = torch.Generator().manual_seed(seed)
    for dim in torch.randperm(D, generator=gen)[:4].tolist():
        q[..., dim] *= 8
        at = torch.from_numpy(places()[0][:, dim]).to(cache.storage.device)
        keys = cache.storage[0, 0]
        byte = keys[..., at]
        # the finite ones in the largest binade: 256 .. 448 of their unit
        keys[..., at] = torch.where((byte & 0x7F) == 0x7F, byte, byte & 0x86 | 0x78).to(torch.uint8)
    check(gpu, cache, q, table, lens, 1.0)
