"""Constrained logits (kernels.constrain_logits) against the definition in
float64, value by value, and the tokens against the returned logits."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from leanstack_amd import kernels

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
FP32, BF16 = torch.float32, torch.bfloat16


def _request(m, v, dtype, length, bias, mask, seed=0, penalties=True):
    """Arguments on the CPU: random tokens (some outside the vocabulary), lengths from 0 to all."""
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(m, v, generator=g) * 3).to(dtype)
    kw = {}
    if length is not None:
        kw["history"] = torch.randint(-2, v + 2, (m, length), generator=g, dtype=torch.int32)
        kw["history"][:, ::3] = kw["history"][:, :1].clone()  # one token many times
        kw["history_lens"] = torch.randint(0, length + 1, (m,), generator=g, dtype=torch.int32)
        kw["history_lens"][:1] = length
        kw["prompt_lens"] = (kw["history_lens"] * torch.rand(m, generator=g)).int()
        if penalties:
            kw["repetition"] = torch.rand(m, generator=g) + 0.5
            kw["frequency"] = torch.rand(m, generator=g) - 0.2
            kw["presence"] = torch.rand(m, generator=g) - 0.2
    if bias:
        kw["bias_ids"] = torch.stack([torch.randperm(v + 4, generator=g)[:bias] - 2 for _ in range(m)]).int()
        kw["bias_values"] = torch.randn(m, bias, generator=g) * 4
    if mask:
        kw["allowed"] = torch.randint(-2**31, 2**31, (m, (v + 31) // 32), generator=g, dtype=torch.int64).int()
    return logits, kw


def _oracle(logits, history=None, history_lens=None, prompt_lens=None, repetition=None, frequency=None, presence=None,
            bias_ids=None, bias_values=None, allowed=None):
    """float64 values, and a bound on what fp32 steps and the final rounding may add.

    A step rounds by at most half an fp32 step, 2^-24 of its result, and later
    steps carry an earlier error on as it is: over the at most five steps (rho,
    alpha_f c, two differences, the bias) that is 2^-24 of the sum of the steps'
    magnitudes, doubled for the errors' own roundings."""
    z = logits.double().numpy().copy()
    m, v = z.shape
    steps = np.zeros_like(z)
    for r in range(m):
        if history is not None:
            n = int(history_lens[r]) if history_lens is not None else history.shape[1]
            n = min(max(n, 0), history.shape[1])
            past = history[r, :n].numpy()
            keep = (past >= 0) & (past < v)
            p = int(prompt_lens[r]) if prompt_lens is not None else 0
            rho = float(repetition[r]) if repetition is not None else 1.0
            seen = np.unique(past[keep])
            z[r, seen] = np.where(z[r, seen] > 0, z[r, seen] / rho, z[r, seen] * rho)
            steps[r, seen] += np.abs(z[r, seen])
            answer = past[max(p, 0):][keep[max(p, 0):]]
            tokens, count = np.unique(answer, return_counts=True)
            af = float(frequency[r]) if frequency is not None else 0.0
            ap = float(presence[r]) if presence is not None else 0.0
            z[r, tokens] -= af * count
            steps[r, tokens] += np.abs(af * count) + np.abs(z[r, tokens])
            z[r, tokens] -= ap
            steps[r, tokens] += np.abs(z[r, tokens])
        if bias_ids is not None:
            last = {int(t): float(b) for t, b in zip(bias_ids[r], bias_values[r]) if 0 <= int(t) < v}
            for t, b in last.items():
                z[r, t] += b
                steps[r, t] += abs(z[r, t])
        if allowed is not None:
            at = np.arange(v)
            words = allowed[r].numpy().view(np.uint32)
            z[r, (words[at >> 5] >> (at & 31).astype(np.uint32)) & 1 == 0] = -math.inf
    fine = np.isfinite(z)
    bound = steps * 2.0 ** -23 + np.where(fine, np.abs(z), 0) * (torch.finfo(logits.dtype).eps / 2) * (1 + 2.0 ** -20)
    # below the type's normal range a rounding is half of its smallest number
    return z, bound + 2.0 ** -133


def _check(got, tokens, z, bound):
    got = got.cpu().double().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(z))
    special = ~np.isfinite(z) & ~np.isnan(z)
    assert np.array_equal(got[special], z[special])
    fine = np.isfinite(z)
    assert (np.abs(got[fine] - z[fine]) <= bound[fine]).all()
    for r, token in enumerate(tokens.tolist()):
        expect = int(np.argmax(got[r]))  # the first of equal values; NaN before all
        assert token == (-1 if got[r][expect] == -math.inf else expect), f"row {r}"


def _run(logits, kw, **more):
    return kernels.constrain_logits(logits.to(DEV), **{k: t.to(DEV) for k, t in kw.items()}, **more)


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("m,v,length,bias,mask", [
    (1, 1, 1, 1, True), (2, 31, 5, 3, True), (3, 33, 40, 0, True), (1, 64, None, 7, False), (4, 1003, 100, 20, True),
    (1, 16384, 17, 0, False), (700, 130, 9, 2, True), (1, 16385, 1000, 1, True), (600, 16320, 50, 2, True), (600, 10176, 70, 2, True), (1500, 20353, 70, 2, True),
    (520, 16321, 50, 0, True), (5, 50257, 300, 1023, True),
    (2, 151936, 4000, 300, True), (64, 20001, 600, 0, False), (600, 33001, 3, 0, True), (3, 4099, None, 0, True),
    (3, 4099, None, 0, False),
])
def test_constrain(gpu, dtype, m, v, length, bias, mask):
    logits, kw = _request(m, v, dtype, length, min(bias, v), mask, seed=v + m)
    got, tokens = _run(logits, kw)
    assert got.dtype == dtype and tokens.dtype == torch.long and tokens.shape == (m,)
    _check(got, tokens, *_oracle(logits, **kw))


def test_defaults_and_lengths_out_of_range(gpu):
    """Without lengths the whole history counts, all of it the answer's; lengths
    outside [0, L] are taken at the ends; without penalties a history changes nothing."""
    logits, kw = _request(3, 1000, FP32, 60, 0, False, seed=1)
    for drop in (("history_lens",), ("prompt_lens",), ("history_lens", "prompt_lens"), ("frequency", "presence"),
                 ("repetition",)):
        some = {k: t for k, t in kw.items() if k not in drop}
        _check(*_run(logits, some), *_oracle(logits, **some))
    got, _ = _run(logits, {k: kw[k] for k in ("history", "history_lens", "prompt_lens")})
    assert torch.equal(got.cpu(), logits)
    far = dict(kw, history_lens=torch.tensor([-5, 10_000, 2**31 - 1], dtype=torch.int32),
               prompt_lens=torch.tensor([-3, 20_000, -2**31], dtype=torch.int32))
    _check(*_run(logits, far), *_oracle(logits, **far))


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_rows_without_a_candidate_and_special_values(gpu, dtype):
    """Nothing allowed: -1.  NaN and infinities where the mask forbids them change
    nothing; where it does not, they go by the formula and NaN is chosen first."""
    v = 5000
    logits, kw = _request(6, v, dtype, 50, 4, True, seed=3)
    kw["allowed"][0] = 0                       # nothing
    kw["allowed"][1] = 0
    kw["allowed"][1, 40] = 1 << 3              # one token
    kw["allowed"][2:] = -1
    bits = torch.arange(v)
    shut = (kw["allowed"][1][bits // 32] >> (bits % 32) & 1) == 0
    logits[0] = math.nan
    logits[1, shut] = math.inf
    logits[1, 7] = math.nan
    logits[2, 4321] = math.nan
    logits[2, 99] = math.inf
    logits[3] = -math.inf                      # allowed, and no candidate
    logits[3, 0], kw["history"][3] = -math.inf, 0
    logits[4] = 0.0
    logits[4, 10:20] = -0.0
    kw["history"][4], kw["bias_ids"][4] = -1, -1
    logits[5] = torch.finfo(dtype).min         # masks of the type's lowest value given as logits
    logits[5, 4999] = torch.finfo(dtype).min / 2
    got, tokens = _run(logits, kw)
    z, bound = _oracle(logits, **kw)
    if dtype is BF16:  # the lowest value less a penalty, or times rho, may round to -inf
        z[5], bound[5] = got[5].cpu().double().numpy(), 1
    else:
        z[5] = np.where(np.abs(z[5]) > torch.finfo(dtype).max, -math.inf, z[5])
    _check(got, tokens, z, bound)
    assert tokens.tolist()[:5] == [-1, 40 * 32 + 3, 4321, -1, 0]


def test_several_biases_for_one_token(gpu):
    logits, kw = _request(2, 3001, FP32, None, 6, False, seed=4)
    kw["bias_ids"][:] = torch.tensor([[5, 9, 5, 9, 5, 7], [3000, 3000, 3000, 0, 3001, -1]])
    got, tokens = _run(logits, kw)
    _check(got, tokens, *_oracle(logits, **kw))
    assert torch.equal(got, _run(logits, kw)[0])


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_strides_alignment_and_in_place(gpu, dtype):
    """Rows of a wider tensor, columns apart, an output at any alignment, the
    logits themselves: the same values; what lies around the output is left."""
    m, v = 5, 4003
    logits, kw = _request(m, v, dtype, 80, 5, True, seed=5)
    expect, tokens = _run(logits, kw)
    dkw = {k: t.to(DEV) for k, t in kw.items()}
    wide = torch.full((m, v + 13), 1e4, dtype=dtype, device=DEV)
    wide[:, 3:3 + v] = logits.to(DEV)
    base = logits.to(DEV)
    forms = [wide[:, 3:3 + v], base.t().contiguous().t(), base.repeat_interleave(2, 1)[:, ::2]]
    for form in forms:
        got, t = kernels.constrain_logits(form, **dkw)
        assert torch.equal(got.view(torch.uint8), expect.view(torch.uint8)) and torch.equal(t, tokens)
    lists = dict(dkw, history=torch.cat((dkw["history"], dkw["history"]), 1)[:, :80],
                 allowed=torch.cat((dkw["allowed"], dkw["allowed"]), 1)[:, :dkw["allowed"].shape[1]])
    assert torch.equal(kernels.constrain_logits(base, **lists)[0].view(torch.uint8), expect.view(torch.uint8))
    for shift in range(1, 9):
        room = torch.full((m * v + 24,), 7.0, dtype=dtype, device=DEV)
        out = room[shift:shift + m * v].view(m, v)
        got, t = kernels.constrain_logits(base, **dkw, out=out)
        assert got is out and torch.equal(out.view(torch.uint8), expect.view(torch.uint8)) and torch.equal(t, tokens)
        assert bool((room[:shift] == 7).all()) and bool((room[shift + m * v:] == 7).all())
    got, t = kernels.constrain_logits(base, **dkw, out=base)
    assert got is base and torch.equal(base.view(torch.uint8), expect.view(torch.uint8)) and torch.equal(t, tokens)
    one = wide[1:2, 3:3 + v]  # one row of the wider tensor is contiguous
    got, _ = kernels.constrain_logits(one, **{k: x[1:2] for k, x in dkw.items()}, out=one)
    assert torch.equal(wide[1, 3:3 + v].view(torch.uint8), expect[1].view(torch.uint8))
    assert bool((wide[:, :3] == torch.tensor(1e4, dtype=dtype)).all())  # what lies around the row is left


def test_empty_calls(gpu):
    got, tokens = kernels.constrain_logits(torch.empty((0, 100), device=DEV))
    assert got.shape == (0, 100) and tokens.shape == (0,)
    logits, _ = _request(2, 100, FP32, None, 0, False)
    none = dict(history=torch.empty((2, 0), dtype=torch.int32), bias_ids=torch.empty((2, 0), dtype=torch.int32),
                bias_values=torch.empty((2, 0)), repetition=torch.full((2,), 2.0))
    got, tokens = _run(logits, none)
    assert torch.equal(got.cpu(), logits) and torch.equal(tokens.cpu(), logits.argmax(1))


def test_captured_and_on_two_streams(gpu):
    """A captured call follows lengths, lists and logits as they are at each
    replay; calls on two streams at once do not share anything."""
    logits, kw = _request(4, 30001, FP32, 500, 30, True, seed=6)
    later, kw2 = _request(4, 30001, FP32, 500, 30, True, seed=7)
    dl, dk = logits.to(DEV), {k: t.to(DEV) for k, t in kw.items()}
    kernels.constrain_logits(dl, **dk)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, kernels.constrain_logits(dl, **dk)))
    for src, lists in ((logits, kw), (later, kw2), (logits, kw2), (later, kw)):
        dl.copy_(src)
        for k, t in dk.items():
            t.copy_(lists[k])
        expect, tokens = kernels.constrain_logits(dl, **dk)
        for graph, (out, t) in graphs:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, expect) and torch.equal(t, tokens)
    a, b = _run(logits, kw), _run(later, kw2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    results = []
    for _ in range(4):
        for stream, (src, lists) in zip(streams, ((dl, dk), (later.to(DEV), {k: t.to(DEV) for k, t in kw2.items()}))):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                results.append(kernels.constrain_logits(src, **lists))
    torch.cuda.synchronize()
    dl_expect = kernels.constrain_logits(dl, **dk)
    for i, (out, t) in enumerate(results):
        expect = b if i % 2 else dl_expect
        assert torch.equal(out, expect[0]) and torch.equal(t, expect[1])
    assert not torch.equal(a[0], b[0])
