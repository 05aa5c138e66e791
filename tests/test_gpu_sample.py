"""Sampled tokens on the GPU against their definition in 64 bits."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from leanstack_amd import kernels

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** 44


def reference(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob) of one row, float64 numpy, by sorting."""
    if np.isnan(row).any() or row.max() == -np.inf:
        return -1, math.nan
    order = np.lexsort((np.arange(len(row)), -row))
    if not temperature > 0:
        return int(order[0]), 0.0
    with np.errstate(invalid="ignore"):
        z = np.where(row == row.max(), 0.0, (row - row.max()) / temperature)
    weight = np.rint(np.exp(z) * UNIT).astype(np.int64)
    kept = order[:top_k] if top_k > 0 else order
    if min_p > 0:
        kept = kept[weight[kept] >= min(min_p, 1.0) * UNIT]
    if top_p < 1:
        before = np.cumsum(weight[kept]) - weight[kept]
        keep = before.astype(np.float64) < top_p * float(weight[kept].sum())
        keep[0] = True
        kept = kept[keep]
    kept = np.sort(kept)
    sums = np.cumsum(weight[kept])
    total = int(sums[-1])
    u = min(max(u, 0.0), 1.0) if u == u else 0.0
    target = min(int(u * float(total)), total - 1)
    token = int(kept[np.searchsorted(sums, target, "right")])
    return token, math.log(int(weight[token]) / total)


def run(gpu, logits, u, **options):
    """Tokens and logprobs of the kernel, checked against the definition row by row."""
    m = logits.shape[0]
    dtypes = dict(top_k=torch.int32)
    given = {name: None if value is None else torch.tensor(value, dtype=dtypes.get(name, torch.float32), device=gpu)
             for name, value in options.items()}
    uniforms = torch.tensor(u, dtype=torch.float32, device=gpu)
    tokens, logs = kernels.sample_logits(logits.to(gpu), uniforms, **given)
    assert tokens.dtype is torch.long and logs.dtype is torch.float32 and tokens.shape == logs.shape == (m,)
    rows = logits.double().numpy()
    per_row = {name: value.cpu().double().tolist() for name, value in given.items() if value is not None}
    for i in range(m):
        args = {name: int(value[i]) if name == "top_k" else value[i] for name, value in per_row.items()}
        token, log = reference(rows[i], float(uniforms[i]), **args)
        assert int(tokens[i]) == token, f"row {i} of {m}: {int(tokens[i])}, not {token} ({args}, u {float(uniforms[i])})"
        got = float(logs[i])
        # one rounding to fp32 (2^-24) and weights that are off by a unit of 2^-44
        assert (math.isnan(got) and math.isnan(log)) or abs(got - log) <= 2.0 ** -23 * abs(log) + 2.0 ** -40 * math.exp(-log) \
            or got == log, f"row {i}: {got}, not {log}"
    return tokens.cpu(), logs.cpu()


def logits_of(m, v, seed, std=3.0, dtype=torch.float32):
    return (torch.randn((m, v), generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def uniforms_of(m, seed):
    return torch.rand((m,), generator=torch.Generator().manual_seed(seed)).tolist()


OPTIONS = [
    {}, dict(temperature=0.7), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.05), dict(temperature=1.3, top_k=40, top_p=0.95),
    dict(top_k=1000, top_p=0.8, min_p=0.01), dict(top_p=0.5, min_p=0.001), dict(top_k=1), dict(temperature=0.0, top_k=5, top_p=0.3),
    dict(temperature=5.0, top_p=0.999), dict(temperature=50.0, top_k=2000),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 2, 63, 64, 65, 1000, 1003, 4097, 32000, 50257, 151936])
def test_options(gpu, v, dtype):
    for i, options in enumerate(OPTIONS):
        m = 3
        run(gpu, logits_of(m, v, seed=v + i, dtype=dtype), uniforms_of(m, seed=i), **{k: [x] * m for k, x in options.items()})


@pytest.mark.parametrize("m", [1, 2, 7, 64, 130, 300])
def test_rows_of_their_own(gpu, m):
    """Every row with its own options, greedy ones among them."""
    rng = np.random.default_rng(m)
    v = 5003
    run(gpu, logits_of(m, v, seed=m), uniforms_of(m, seed=m + 1), temperature=rng.choice([0.0, 0.5, 1.0, 2.0], m).tolist(),
        top_k=rng.choice([0, -1, 1, 3, 100, 4000, 5003, 1 << 30], m).tolist(),
        top_p=rng.choice([0.0, -1.0, 0.1, 0.9, 1.0, 2.0], m).tolist(), min_p=rng.choice([0.0, -0.5, 1e-4, 0.1, 1.0, 3.0], m).tolist())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [500, 9001])
@pytest.mark.parametrize("temperature", [1e37, 1e38, 3e38, math.inf])
def test_values_further_apart_than_the_largest_number(gpu, temperature, v, dtype):
    """Differences that overflow in 32 bits, at temperatures that make them small."""
    logits = logits_of(3, v, seed=21, std=1.0, dtype=dtype).clamp(-3.3, 3.3) * 1e38
    if math.isfinite(temperature):
        logits[2, ::7] = -math.inf
    for i, options in enumerate(({}, dict(top_k=40), dict(top_k=400, top_p=0.7), dict(top_p=0.6), dict(min_p=0.01), dict(min_p=0.9))):
        run(gpu, logits, uniforms_of(3, seed=22 + i), temperature=[temperature] * 3, **{k: [x] * 3 for k, x in options.items()})


@pytest.mark.parametrize("std", [0.0, 1e-6, 0.01, 30.0, 1e4, 1e30])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_flat_and_steep(gpu, std, dtype):
    """All logits equal or nearly so (the whole row in a bin), and so far apart that one token has all the weight."""
    m, v = 4, 20011
    logits = logits_of(m, v, seed=3, std=std, dtype=dtype)
    for i, options in enumerate(({}, dict(top_k=7000), dict(top_p=0.3), dict(top_k=9000, top_p=0.7, min_p=0.2), dict(min_p=1.0),
                                 dict(temperature=1e-3, top_p=0.9), dict(temperature=1e-30), dict(temperature=1e30, top_k=11))):
        run(gpu, logits, uniforms_of(m, seed=4 + i), **{k: [x] * m for k, x in options.items()})


def test_ties_take_the_lower_index(gpu):
    logits = torch.zeros((1, 3001))
    logits[0, 2999] = 1.0
    for k, u, want in ((1, 0.9, 2999), (2, 0.0, 0), (2, 0.999, 2999), (3, 0.3, 1), (4, 0.99, 2999)):
        tokens, _ = run(gpu, logits, [u], top_k=[k])
        assert int(tokens[0]) == want
    tokens, _ = run(gpu, torch.zeros((1, 100)), [0.5], top_p=[0.5])  # the first fifty exactly
    assert int(tokens[0]) == 25
    tokens, _ = run(gpu, torch.zeros((1, 100)), [0.999], top_p=[0.5])
    assert int(tokens[0]) == 49


def test_minus_zero_is_zero(gpu):
    logits = torch.full((1, 64), -1.0)
    logits[0, 5], logits[0, 9] = -0.0, 0.0
    tokens, _ = run(gpu, logits, [0.0], top_k=[1])
    assert int(tokens[0]) == 5


@pytest.mark.parametrize("u", [0.0, -0.0, -1.0, 1.0, 2.0, math.nan, math.inf, 1 - 2.0 ** -24, 2.0 ** -149])
def test_ends_of_the_random_number(gpu, u):
    logits = torch.full((1, 500), -math.inf)
    logits[0, 7], logits[0, 300], logits[0, 450] = 1.0, 2.0, 0.5
    tokens, _ = run(gpu, logits, [u])
    assert int(tokens[0]) == (450 if u >= 1 - 2.0 ** -24 else 7)


def test_masked_infinite_and_nan_rows(gpu):
    logits = logits_of(8, 999, seed=6)
    logits[0, :] = -math.inf
    logits[1, 500] = math.nan
    logits[2, :] = -math.inf
    logits[2, 998] = -3e38
    logits[3, 10], logits[3, 20] = math.inf, math.inf
    logits[4, 1:] = -math.inf
    logits[5, :] = math.nan
    logits[6, 0], logits[6, 1] = math.inf, math.nan
    logits[7, 3:] = torch.finfo(torch.float32).min
    for options in ({}, dict(top_k=[3] * 8), dict(top_p=[0.9] * 8, min_p=[0.1] * 8), dict(temperature=[0.0] * 8)):
        tokens, logs = run(gpu, logits, uniforms_of(8, seed=7), **options)
        assert tokens[[0, 1, 5, 6]].tolist() == [-1] * 4 and bool(torch.isnan(logs[[0, 1, 5, 6]]).all())
        assert tokens[[2, 4]].tolist() == [998, 0] and tokens[3] in (10, 20)


def test_options_that_are_nan(gpu):
    logits = logits_of(3, 300, seed=8)
    tokens, _ = kernels.sample_logits(logits.to(gpu), torch.full((3,), 0.7, device=gpu),
                                      temperature=torch.tensor([math.nan, 1.0, 1.0], device=gpu),
                                      top_p=torch.tensor([1.0, math.nan, 1.0], device=gpu),
                                      min_p=torch.tensor([0.0, 0.0, math.nan], device=gpu))
    want = [int(logits[0].argmax())] + [reference(logits[i].double().numpy(), float(np.float32(0.7)))[0] for i in (1, 2)]
    assert tokens.tolist() == want


def test_every_token_is_drawn_as_often_as_its_weight_says(gpu):
    """Random numbers on an even grid hit each token within one of its share."""
    m, v = 4096, 37
    logits = logits_of(1, v, seed=9, std=1.0).expand(m, v).contiguous()
    u = ((np.arange(m) + 0.5) / m).astype(np.float32).tolist()
    tokens, logs = run(gpu, logits, u)
    share = torch.softmax(logits[0].double(), -1) * m
    assert bool(((torch.bincount(tokens, minlength=v) - share).abs() <= 1).all())
    assert bool((tokens[1:] >= tokens[:-1]).all())


def test_views(gpu):
    """Rows of a padded vocabulary, rows that do not start on 16 bytes, a transposed one."""
    m, v = 5, 2001
    for dtype in (torch.float32, torch.bfloat16):
        logits = logits_of(m, v, seed=10, dtype=dtype)
        u = torch.tensor(uniforms_of(m, seed=11), device=gpu)
        k = torch.full((m,), 30, dtype=torch.int32, device=gpu)
        want = kernels.sample_logits(logits.to(gpu), u, top_k=k)
        wide = torch.full((m, v + 64), 99.0, dtype=dtype, device=gpu)
        wide[:, 3:3 + v] = logits.to(gpu)
        for same in (wide[:, 3:3 + v], logits.to(gpu).t().contiguous().t()):
            got = kernels.sample_logits(same, u, top_k=k)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_same_result_every_time(gpu):
    logits = logits_of(16, 151936, seed=12).to(gpu)
    u = torch.tensor(uniforms_of(16, seed=13), device=gpu)
    p = torch.full((16,), 0.99, device=gpu)
    want = kernels.sample_logits(logits, u, top_p=p)
    for _ in range(20):
        got = kernels.sample_logits(logits, u, top_p=p)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured(gpu):
    """Replays follow everything on the device, beside eager calls on the same stream."""
    m, v = 6, 32000
    logits, u = logits_of(m, v, seed=14).to(gpu), torch.tensor(uniforms_of(m, seed=15), device=gpu)
    t, k = torch.ones(m, device=gpu), torch.full((m,), 20, dtype=torch.int32, device=gpu)
    p, mp = torch.full((m,), 0.9, device=gpu), torch.zeros(m, device=gpu)
    kernels.sample_logits(logits, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = kernels.sample_logits(logits, u, temperature=t, top_k=k, top_p=p, min_p=mp)
        second = kernels.sample_logits(logits, u)
    for i in range(5):
        logits.copy_(logits_of(m, v, seed=20 + i).to(gpu)), u.copy_(torch.tensor(uniforms_of(m, seed=30 + i)))
        t.fill_(0.5 * i), k.fill_(100 * i), p.fill_(1 - 0.1 * i), mp.fill_(0.01 * i)
        graph.replay()
        eager = kernels.sample_logits(logits, u, temperature=t, top_k=k, top_p=p, min_p=mp)
        other = kernels.sample_logits(logits, u)
        torch.cuda.synchronize()
        for got, want in ((first, eager), (second, other)):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_streams(gpu):
    v = 50257
    fed = [(logits_of(9, v, seed=40 + i).to(gpu), torch.tensor(uniforms_of(9, seed=50 + i), device=gpu)) for i in range(4)]
    k = torch.full((9,), 77, dtype=torch.int32, device=gpu)
    want = [kernels.sample_logits(x, u, top_k=k) for x, u in fed]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[] for _ in fed]
    for _ in range(10):
        for i, (x, u) in enumerate(fed):
            with torch.cuda.stream(streams[i % 2]):
                got[i].append(kernels.sample_logits(x, u, top_k=k))
    torch.cuda.synchronize()
    for i in range(4):
        assert all(torch.equal(a, want[i][0]) and torch.equal(b, want[i][1]) for a, b in got[i])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,v", [(1, 24576), (1, 24583), (2, 32771), (7, 151936), (1, 1 << 19), (1, (1 << 19) - 3), (128, 40003), (170, 24587),
                                 (171, 24587)])
def test_few_rows_without_ranks(gpu, m, v, dtype):
    """Temperature and top-p alone, rows that several workgroups share: every row with its own options, greedy
    ones and ones that top-p leaves alone among them."""
    rng = np.random.default_rng(v)
    logits = logits_of(m, v, seed=v, dtype=dtype)
    temperature = rng.choice([0.0, 0.4, 1.0, 1.7], m).tolist()
    run(gpu, logits, uniforms_of(m, seed=1), temperature=temperature)
    run(gpu, logits, uniforms_of(m, seed=2))
    run(gpu, logits, uniforms_of(m, seed=3), temperature=temperature, top_p=rng.choice([0.0, 0.3, 0.9, 0.999, 1.0, math.nan], m).tolist())
    run(gpu, logits, [0.0, 1.0][: min(m, 2)] + uniforms_of(m, seed=4)[2:], top_p=[0.95] * m)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_where_the_cut_falls_in_sliced_rows(gpu, dtype):
    """Cuts among equal values all over the row (more than are listed, and fewer), in the first and in the last
    slice, rows of one value and rows at odd addresses."""
    v = 65536 + 24
    base = torch.full((6, v + 5), -20.0)
    base[0] = 1.0                              # all equal: no list holds them
    base[1, ::40] = 2.0                        # 1600 equal ones
    base[2, ::9] = 2.0                         # 7000
    base[3, :300] = torch.arange(300) / 100    # in the first slice
    base[4, -300:] = torch.arange(300) / 100   # in the last one
    base[5, ::3] = torch.randn((len(base[5, ::3]),), generator=torch.Generator().manual_seed(5)) * 0.02
    wide = base.to(dtype).to(gpu)
    for at in (0, 1, 3, 5):
        logits = wide[:, at:at + v]
        for i, top_p in enumerate((0.01, 0.5, 0.97, 0.99999)):
            u = uniforms_of(6, seed=50 + i)
            tokens, logs = kernels.sample_logits(logits, torch.tensor(u, device=gpu), top_p=torch.full((6,), top_p, device=gpu))
            rows = logits.double().cpu().numpy()
            for r in range(6):
                token, log = reference(rows[r], float(torch.tensor(u)[r]), top_p=float(torch.tensor(top_p)))
                assert int(tokens[r]) == token, f"row {r} at {at}, top_p {top_p}"
                assert abs(float(logs[r]) - log) <= 2.0 ** -23 * abs(log) + 2.0 ** -40 * math.exp(-log)


@pytest.mark.parametrize("at", [0, 9000, 20000, 32767])
def test_nan_and_infinities_in_sliced_rows(gpu, at):
    """A NaN in any slice, a row of -inf, one value that is not, values of +inf in several slices."""
    v = 32768
    logits = logits_of(5, v, seed=60)
    logits[0, at] = math.nan
    logits[1] = -math.inf
    logits[2] = -math.inf
    logits[2, at] = -3e38
    logits[3, at] = logits[3, 77] = logits[3, 30000] = math.inf
    for options in ({}, dict(top_p=[0.7] * 5), dict(top_p=[0.2] * 5, temperature=[0.0, 0.0, 1.0, 1.0, 0.0])):
        run(gpu, logits, uniforms_of(5, seed=61), **options)


def test_captured_sliced_rows_follow_their_arguments(gpu):
    """Replays with other logits and options, eager calls in between."""
    m, v = 4, 50000
    logits, u = torch.zeros((m, v), device=gpu), torch.zeros(m, device=gpu)
    temperature, top_p = torch.ones(m, device=gpu), torch.ones(m, device=gpu)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        tokens, logs = kernels.sample_logits(logits, u, temperature=temperature, top_p=top_p)
        alone, alone_logs = kernels.sample_logits(logits, u, temperature=temperature)
    rng = np.random.default_rng(70)
    for i in range(5):
        fresh = logits_of(m, v, seed=70 + i)
        options = dict(temperature=rng.choice([0.0, 0.6, 1.2], m).tolist(), top_p=rng.choice([0.2, 0.9, 1.0], m).tolist())
        given = uniforms_of(m, seed=80 + i)
        logits.copy_(fresh), u.copy_(torch.tensor(given))
        temperature.copy_(torch.tensor(options["temperature"])), top_p.copy_(torch.tensor(options["top_p"]))
        graph.replay()
        want = run(gpu, fresh, given, **options)
        assert torch.equal(tokens.cpu(), want[0]) and torch.equal(logs.cpu(), want[1])
        want = run(gpu, fresh, given, temperature=options["temperature"])
        assert torch.equal(alone.cpu(), want[0]) and torch.equal(alone_logs.cpu(), want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,v", [(1, 65536), (1, 131072), (2, 131071), (7, 151936), (1, 1 << 19), (1, (1 << 19) - 3), (170, 65541), (171, 65541)])
def test_few_rows_with_ranks(gpu, m, v, dtype):
    """top-k and min-p on rows that several workgroups share: every row with its own options, some off, some greedy."""
    rng = np.random.default_rng(v + 1)
    logits = logits_of(m, v, seed=v + 1, dtype=dtype)
    temperature = rng.choice([0.0, 0.4, 1.0, 1.7], m).tolist()
    top_k = rng.choice([0, 1, 7, 50, 1000, 2048, 2049, 9000], m).tolist()
    min_p = rng.choice([0.0, 1e-6, 0.03, 0.9, 1.0, math.nan], m).tolist()
    top_p = rng.choice([0.0, 0.3, 0.95, 1.0], m).tolist()
    run(gpu, logits, uniforms_of(m, seed=1), temperature=temperature, top_k=top_k)
    run(gpu, logits, uniforms_of(m, seed=2), temperature=temperature, min_p=min_p)
    run(gpu, logits, uniforms_of(m, seed=3), temperature=temperature, top_k=top_k, min_p=min_p, top_p=top_p)
    run(gpu, logits, uniforms_of(m, seed=4), top_k=[50] * m, top_p=[0.9] * m)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_where_the_ranks_fall_in_sliced_rows(gpu, dtype):
    """The first k among equal values all over the row (more than the lists hold, and fewer), all in one slice, in rows
    at odd addresses; rows of -inf, NaN and +inf."""
    v = 131072 + 24
    base = torch.full((8, v + 5), -20.0)
    base[0] = 1.0
    base[1, ::80] = 2.0
    base[2, ::9] = 2.0
    base[3, :300] = torch.arange(300) / 100
    base[4, -300:] = torch.arange(300) / 100
    base[5] = -math.inf
    base[5, 40000] = -5.0
    base[6, 50000] = math.nan
    base[7, 20000:60000:13000] = math.inf
    wide = base.to(dtype).to(gpu)
    for at in (0, 1, 3, 5):
        logits = wide[:, at:at + v]
        rows = logits.double().cpu().numpy()
        for i, (k, min_p, top_p) in enumerate(((1, 0.0, 1.0), (40, 0.0, 0.9), (1700, 0.0, 0.5), (100, 0.02, 1.0), (0, 0.3, 1.0), (2000, 1e-12, 0.99))):
            u = uniforms_of(8, seed=90 + i)
            full = [torch.full((8,), x, device=gpu) for x in (k, min_p, top_p)]
            tokens, logs = kernels.sample_logits(logits, torch.tensor(u, device=gpu), top_k=full[0].int(), min_p=full[1], top_p=full[2])
            for r in range(8):
                token, log = reference(rows[r], float(torch.tensor(u)[r]), top_k=k, min_p=float(full[1][r]), top_p=float(full[2][r]))
                assert int(tokens[r]) == token, f"row {r} at {at}, top_k {k}, min_p {min_p}, top_p {top_p}"
                assert math.isnan(log) and math.isnan(float(logs[r])) \
                    or abs(float(logs[r]) - log) <= 2.0 ** -23 * abs(log) + 2.0 ** -40 * math.exp(-log)


def test_captured_ranked_rows_follow_their_arguments(gpu):
    m, v = 5, 66000
    logits, u = torch.zeros((m, v), device=gpu), torch.zeros(m, device=gpu)
    given = dict(temperature=torch.ones(m, device=gpu), top_k=torch.ones(m, dtype=torch.int32, device=gpu), top_p=torch.ones(m, device=gpu),
                 min_p=torch.zeros(m, device=gpu))
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        tokens, logs = kernels.sample_logits(logits, u, **given)
    rng = np.random.default_rng(71)
    for i in range(5):
        fresh = logits_of(m, v, seed=170 + i)
        options = dict(temperature=rng.choice([0.0, 0.6, 1.2], m).tolist(), top_k=rng.choice([0, 3, 60, 900], m).tolist(),
                       top_p=rng.choice([0.2, 0.9, 1.0], m).tolist(), min_p=rng.choice([0.0, 0.05], m).tolist())
        draw = uniforms_of(m, seed=180 + i)
        logits.copy_(fresh), u.copy_(torch.tensor(draw))
        for name, value in options.items():
            given[name].copy_(torch.tensor(value))
        graph.replay()
        want = run(gpu, fresh, draw, **options)
        assert torch.equal(tokens.cpu(), want[0]) and torch.equal(logs.cpu(), want[1])
