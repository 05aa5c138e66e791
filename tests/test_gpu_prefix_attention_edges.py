"""Attention over a shared prefix at its edges: batches that have nothing to attend,
infinities in rows that weigh nothing."""

from __future__ import annotations

import math

import pytest
import torch

from leanstack_amd import kernels
from tests import test_gpu_prefix_attention as attention_of

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
D = 128
SCALE = D ** -0.5


@pytest.mark.parametrize("b,t,n_q,n_kv", [(32, 1, 32, 8), (33, 1, 32, 8), (300, 1, 4, 1), (64, 1, 32, 8), (9, 40, 32, 8)])
def test_large_batches_without_any_row(gpu, b, t, n_q, n_kv):
    """No prefix and no room for own rows: zeros, however many requests there are."""
    q, pk, pv, k, v, _ = attention_of._request(b, t, n_q, n_kv, 0, 1)
    none = k[:, :, :0]
    for lens in (torch.zeros(b, dtype=torch.int32, device=DEV), torch.full((b,), 7, dtype=torch.int32, device=DEV)):
        out = torch.full((b, t, n_q * D), 9.0, device=DEV).bfloat16()
        assert kernels.shared_prefix_attention(q, pk, pv, none, v[:, :, :0], lens, SCALE, out=out) is out
        assert not bool(out.any())


@pytest.mark.parametrize("prefix,b", [(100, 2), (1000, 2), (1000, 40), (1000, 60)])
@pytest.mark.parametrize("t", [1, 2, 5])
def test_an_infinity_of_no_weight(gpu, prefix, b, t):
    """A row that scores -inf weighs e^-inf = 0, and 0 times an infinite value is NaN, also
    where only some of the queries see the row; the others do not meet it."""
    q, pk, pv, k, v, lens = attention_of._request(b, t, 8, 2, prefix, 50, seed=11)
    lens[0] = 33
    q[0] = q[0].abs() + 0.1
    k[0, :, :33], v[0, :, :33] = 0.25, 0.5
    k[0, 0, 32] = -math.inf             # seen by the last query alone; heads 0..3
    base = kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE)
    v[0, 0, 32, 5], v[0, 0, 32, 70], v[0, 1, 32, 6] = math.inf, -math.inf, math.inf
    got = kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE)
    assert torch.equal(got[1:].nan_to_num(7.0), base[1:].nan_to_num(7.0)) and torch.equal(got[0, : t - 1], base[0, : t - 1])
    heads, old = got[0, t - 1].view(8, D), base[0, t - 1].view(8, D)
    assert bool(heads[:4, [5, 70]].isnan().all()) and bool((heads[4:, 6] == math.inf).all())
    rest = torch.ones((8, D), dtype=torch.bool, device=DEV)
    rest[:4, [5, 70]], rest[4:, 6] = False, False
    assert torch.equal(heads[rest], old[rest])
