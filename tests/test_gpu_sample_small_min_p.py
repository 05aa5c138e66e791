"""min_p of a few units of 2^-44: weights are rounded before they are compared, so what is
up to half a unit below min_p is kept, on every route."""

from __future__ import annotations

import math

import pytest
import torch

from test_gpu_sample import reference, run

pytestmark = pytest.mark.gpu

TOP = 3.0


def rounded_up(dtype, least: int):
    """(x, units): the lowest logit of the type whose weight beside TOP rounds up, by 0.1 or more, to `least` units of 2^-44 or more."""
    for i in range(8192):
        x = float(torch.tensor(TOP + math.log((least - 0.5) * 2.0 ** -44) + i * 2.0 ** -10).to(dtype))
        weight = math.exp(x - TOP) * 2.0 ** 44
        units = round(weight)
        if units >= least and 0.1 < units - weight < 0.49:
            return x, units
    raise AssertionError


def without_weight(m, v):
    """Rows of which no value weighs beside TOP, and no more than a few in a thousand beside their neighbours."""
    logits = torch.full((m, v), -1e4)
    logits[:, ::500] = -100.0
    return logits


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [1000, 20011, 151936])  # short rows, whole rows, rows in slices
@pytest.mark.parametrize("least", [1, 2, 3, 5, 9, 17, 40])
@pytest.mark.parametrize("top_k", [0, 3])
def test_a_weight_that_rounds_up_to_min_p_is_kept(gpu, v, dtype, least, top_k):
    x, units = rounded_up(dtype, least)
    min_p = units * 2.0 ** -44
    logits = without_weight(2, v).to(dtype)
    logits[:, 300], logits[:, 500] = TOP, TOP - 1
    logits[0, v - 1], logits[1, 0] = x, x
    options = dict(min_p=[min_p] * 2) | (dict(top_k=[top_k] * 2) if top_k else {})
    tokens, _ = run(gpu, logits, [1.0, 0.0], **options)
    assert tokens.tolist() == [v - 1, 0]


@pytest.mark.parametrize("v", [6000, 20011, 151936])
def test_more_such_tokens_than_a_list_holds(gpu, v):
    """All of a row but its maximum weigh 1.6 units, or 1.4: kept, or not, as one."""
    for units, kept in ((1.6, True), (1.4, False)):
        logits = torch.full((1, v), TOP + math.log(units * 2.0 ** -44))
        logits[0, 100] = TOP
        u = 1.0
        tokens, _ = run(gpu, logits, [u], min_p=[2.0 ** -43])
        assert int(tokens[0]) == (v - 1 if kept else 100)


@pytest.mark.parametrize("v", [3000, 30000, 151936])
@pytest.mark.parametrize("min_p", [2.0 ** -44, 2.0 ** -45, 1e-14, 2.0 ** -149, 2.0 ** -43 * 1.25, 2.0 ** -40 * 0.99])
def test_min_p_between_whole_units(gpu, min_p, v):
    """Logits in steps of a hundredth over the last octaves, some kept and some not."""
    row = without_weight(1, v)[0]
    row[:1500] = TOP - 40 * math.log(2) - torch.arange(1500) * 0.01
    row[700] = TOP
    rows = row[None].repeat(3, 1)
    run(gpu, rows, [0.0, 1.0 - 2.0 ** -24, 1.0], min_p=[min_p] * 3)
    run(gpu, rows.flip(1).contiguous(), [0.0, 1.0 - 2.0 ** -24, 1.0], min_p=[min_p] * 3)


def test_the_reference_keeps_them():
    row = torch.full((10,), -100.0).double().numpy()
    row[3], row[9] = TOP, TOP + math.log(1.6 * 2.0 ** -44)
    assert reference(row, 1.0, min_p=2.0 ** -43)[0] == 9 and reference(row, 1.0, min_p=2.0 ** -42)[0] == 3
