"""Attention over a shared prefix at its edges: batches that have nothing to attend,
infinities in rows that weigh nothing, scores of any finite size."""

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


CASES = [(3, 1, 8, 2, 64, 50), (3, 4, 8, 2, 100, 300), (3, 1, 8, 2, 1500, 300), (3, 5, 8, 2, 1500, 300), (50, 1, 8, 2, 1500, 100),
         (20, 4, 8, 2, 700, 400)]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("signs", ["both", "negative", "positive"])
def test_scores_of_any_size(gpu, case, signs):
    """Scores are powers of two from 2^10 to 2^110, times one factor, and their negatives, so
    that the rows of the largest share a query's weight evenly and the others' is below
    2^-60: the result is the mean of their values, however large the scores are (the
    factor's 16 bits leave the exponents inexact in fp32).

    The mean's weights are equal, the sums of n values lose n fp32 steps, 2^-23 of the
    largest, and the output is rounded once, by 2^-8."""
    b, t, n_q, n_kv, prefix, rows = case
    gen = torch.Generator(device=DEV).manual_seed(sum(case))
    q, pk, pv, k, v, lens = attention_of._request(*case, seed=12)
    k.nan_to_num_(0.0), v.nan_to_num_(0.0)

    def keys(x, low, high):
        """A power of two times 207 / 128 in each row's first place, most rows at the lower end."""
        size = torch.rand(x.shape[:-1], generator=gen, device=DEV) ** 4 * (high - low)
        sign = torch.randint(0, 2, x.shape[:-1], generator=gen, device=DEV) * 2 - 1
        x.zero_()
        x[..., 0] = 207 / 128 * torch.exp2(low + size.floor()) * (sign if signs == "both" else -1 if signs == "negative" else 1)

    q.zero_()
    q[..., 0] = 179 / 128 * torch.exp2(torch.randint(5, 56, q.shape[:-1], generator=gen, device=DEV).float())
    keys(pk, 5.0, 55.0), keys(k, 5.0, 55.0)
    k[::2] = k[::2].clamp(-64 * 207 / 128, 64 * 207 / 128)          # some requests' own rows are no match for the prefix
    got = kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE).view(b, t, n_q, D).double()
    for i, length in enumerate(lens.tolist()):
        for j in range(t):
            own = max(0, length - (t - 1 - j))
            for h in range(n_q):
                score = torch.cat((pk[h // (n_q // n_kv), :, 0], k[i, h // (n_q // n_kv), :own, 0])).double()
                values = torch.cat((pv[h // (n_q // n_kv)], v[i, h // (n_q // n_kv), :own])).double()
                top = values[score == score.max()]
                mean = top.mean(0)
                bound = mean.abs() * 2.0 ** -8 + 2 * (len(top) + 80) * 2.0 ** -23 * top.abs().amax(0)
                assert bool(((got[i, j, h] - mean).abs() <= bound).all()), (i, j, h, len(top), float(q[i, h, j, 0] * score.max()))
