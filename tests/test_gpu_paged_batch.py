"""Serving steps of a batch over the paged 8-bit cache with constrained, sampled answers:
prompts, forks, single tokens, verify blocks with rejected drafts, and compaction in
between.  The result of each operator against its definition on the inputs that it was
really given, and captured steps against eager ones."""

from __future__ import annotations

import math
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from leanstack_amd import _lib, kernels
from leanstack_amd.layout import PackedWeight
from leanstack_amd.paged_cache import PagedKVCache
from tests import test_gpu_constrain as constraints_of
from tests import test_gpu_sample as samples_of
from tests.helpers import seeded_normal
from tests.paged_helpers import D, Pool, attention

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
N_Q, N_KV, VOCAB, LAYERS = 8, 2, 2000, 2
H, SCALE = N_Q * D, 128 ** -0.5


class Model:
    """Random weights of attention layers and a head."""

    def __init__(self):
        def packed(n, std, seed):
            return PackedWeight.from_rowmajor(seeded_normal((n, H), std, seed).to(DEV), _lib.LAYOUT_MFMA16X32)

        self.embed = seeded_normal((VOCAB, H), 1.0, 1).to(DEV)
        self.norm = (1 + seeded_normal((H,), 0.1, 2)).to(DEV)
        self.qkv = [packed((N_Q + 2 * N_KV) * D, H ** -0.5, 10 + i) for i in range(LAYERS)]
        self.o = [packed(H, H ** -0.5, 20 + i) for i in range(LAYERS)]
        self.head = packed(VOCAB, 0.1, 30)


class Settings:
    """A batch's constraints and sampling options, and its random numbers."""

    def __init__(self, b):
        with torch.device("cpu"):   # (also under another default device)
            gen = torch.Generator().manual_seed(b)
            self.bias = dict(bias_ids=torch.randint(0, VOCAB, (b, 7), generator=gen).int().to(DEV),
                             bias_values=torch.randn(b, 7, generator=gen).to(DEV),
                             allowed=torch.randint(-2**31, 2**31, (b, (VOCAB + 31) // 32), generator=gen,
                                                   dtype=torch.int64).int().to(DEV))
            pick = torch.arange(b)
            self.options = dict(temperature=torch.tensor([0.0, 0.7, 1.0, 1.5])[pick % 4].to(DEV),
                                top_k=torch.tensor([0, 40, 1000], dtype=torch.int32)[pick % 3].to(DEV),
                                top_p=torch.tensor([0.9, 1.0])[pick // 2 % 2].to(DEV),
                                min_p=torch.tensor([0.0, 0.05, 0.0])[pick % 3].to(DEV))
            self.uniforms = torch.rand((b,), generator=gen).to(DEV)


def step(model, cache, settings, tokens, table, lens, counts=None, seen=None):
    """Sampled tokens and their logprobs behind each request's last row of tokens [B, T]
    (the rows of them that count), which become rows of the cache."""
    b, t = tokens.shape
    hidden = model.embed[tokens]
    for layer in range(LAYERS):
        qkv = kernels.linear(kernels.rmsnorm_rows(hidden, model.norm, 1e-6), model.qkv[layer])
        qkv = qkv.view(b, t, N_Q + 2 * N_KV, D).transpose(1, 2)
        q, k, v = qkv.split([N_Q, N_KV, N_KV], 1)   # (views of the projection's rows)
        before = Pool(cache.storage[layer], cache.exponents[layer]) if seen is not None else None
        kernels.paged_append(cache, layer, k, v, table, lens, counts=counts)
        out = kernels.paged_attention(q, cache, layer, table, lens, SCALE, counts=counts)
        if seen is not None:
            after = Pool(cache.storage[layer], cache.exponents[layer])
            seen.append(("rows", (before, k, v, table, lens, counts), after))
            seen.append(("attention", (after, q, table, lens, counts), out))
        hidden = kernels.linear(out, model.o[layer], epilogue=_lib.EPI_RESIDUAL_ADD, residual=hidden)
    last = torch.full((b,), t, device=DEV) if counts is None else counts
    rows = hidden[torch.arange(b, device=DEV), (last.long() - 1).clamp(min=0)]
    rows = kernels.rmsnorm_rows(rows, model.norm, 1e-6)
    if b <= _lib.DECODE_MAX_M:
        logits = torch.empty((b, VOCAB), device=DEV)
        kernels.lm_head_argmax(rows, model.head, logits_out=logits)
    else:
        logits = kernels.linear(rows, model.head)
    values, greedy = kernels.constrain_logits(logits, **settings.bias)
    token, logprob = kernels.sample_logits(values, settings.uniforms, **settings.options)
    if seen is not None:
        seen.append(("constraints", (logits, settings.bias), (values, greedy)))
        seen.append(("sample", (values, settings.uniforms.clone(), settings.options), (token, logprob)))
    return token, logprob


def listed(x):
    return None if x is None else x.tolist()


def verify(seen):
    for kind, inputs, result in seen:
        if kind == "rows":
            pool, k, v, table, lens, counts = inputs
            pool.append(k.cpu(), v.cpu(), table.tolist(), lens.tolist(), listed(counts))
            assert (pool.exponents == result.exponents).all() and (pool.bytes == result.bytes).all()
        elif kind == "attention":
            pool, q, table, lens, counts = inputs
            want, bound = attention(pool, q.cpu(), table.tolist(), lens.tolist(), SCALE, listed(counts))
            assert bool(((result.cpu().double().view(want.shape) - want).abs() <= bound).all())
        elif kind == "constraints":
            logits, settings = inputs
            z, bound = constraints_of._oracle(logits.cpu(), **{name: x.cpu() for name, x in settings.items()})
            constraints_of._check(result[0], result[1], z, bound)
        else:
            values, uniforms, options = inputs
            per_row = {name: x.cpu().double().tolist() for name, x in options.items()}
            for i, row in enumerate(values.cpu().double().numpy()):
                args = {name: int(x[i]) if name == "top_k" else x[i] for name, x in per_row.items()}
                token, log = samples_of.reference(row, float(uniforms[i]), **args)
                assert int(result[0][i]) == token
                # one rounding to fp32 (2^-24) and weights that are off by a unit of 2^-44
                assert abs(float(result[1][i]) - log) <= 2.0 ** -23 * abs(log) + 2.0 ** -40 * math.exp(-log)


def prompts(model, cache, lengths, seen=None):
    """Requests with prompts of these lengths in the cache, written by one padded step."""
    requests = [cache.open() for _ in lengths]
    cache.reserve(requests, lengths)
    table, lens = cache.batch(requests, lengths)
    tokens = torch.arange(len(lengths) * max(lengths), device=DEV).view(len(lengths), -1) * 31 % VOCAB
    token, _ = step(model, cache, Settings(len(lengths)), tokens, table, lens,
                    torch.tensor(lengths, dtype=torch.int32, device=DEV), seen)
    cache.advance(requests, lengths)
    return requests, token


@pytest.mark.parametrize("page_rows,lengths", [(16, [5, 37, 1, 16]), (64, [300, 64, 129]), (32, [1300, 7])])
def test_a_batch_from_prompts_to_answers(gpu, page_rows, lengths):
    """Prompts, a fork of each, single tokens, verify blocks whose drafts are partly
    rejected, a request that ends, and compaction: every call against its definition."""
    model, seen = Model(), []
    cache = PagedKVCache(LAYERS, N_KV, 3 * sum(-(-(n + 40) // page_rows) for n in lengths), page_rows=page_rows, device=DEV)
    requests, token = prompts(model, cache, lengths, seen)
    requests = requests + [cache.fork(r) for r in requests]
    b = len(requests)
    token = token.repeat(2)
    settings = Settings(b)
    for at in range(6):
        draft = [4, 1, 3, 2, 4, 1][at]
        counts = [1 + (i + at) % draft for i in range(b)]
        cache.reserve(requests, counts)
        table, lens = cache.batch(requests, counts)
        tokens = (token.clamp(min=0)[:, None] + torch.arange(draft, device=DEV)) % VOCAB
        settings.uniforms.copy_(torch.rand((b,), generator=torch.Generator().manual_seed(at)))
        token, _ = step(model, cache, settings, tokens, table, lens,
                        None if draft == 1 else torch.tensor(counts, dtype=torch.int32, device=DEV), seen)
        cache.advance(requests, counts)
        for i, r in enumerate(requests):   # (some drafts are rejected)
            cache.truncate(r, r.rows - counts[i] // 2)
        if at == 2:
            cache.close(requests.pop(0))
            token, b = token[1:].contiguous(), b - 1
            settings = Settings(b)
        if at == 3:
            kept = [cache.storage[:, :, r.pages].clone() for r in requests]
            assert cache.compact() == cache.num_pages - cache.free_pages
            assert all(torch.equal(x, cache.storage[:, :, r.pages]) for x, r in zip(kept, requests))
    verify(seen)
    assert len(seen) == 7 * (2 * LAYERS + 2)


@pytest.mark.parametrize("b,t,width", [(1, 1, 40), (12, 1, 40), (12, 1, 80), (5, 4, 40), (5, 4, 80), (60, 1, 80), (3, 40, 80)])
def test_captured_steps_are_the_eager_ones(gpu, b, t, width):
    """One captured step, replayed with new tables, lengths, random numbers and options:
    what eager steps give, also with pages that moved between the replays.  (A table of
    the same width on both sides: it decides how a call is cut.)"""
    model = Model()
    lengths = [1 + 97 * i % 500 for i in range(b)]
    eager, captured = (PagedKVCache(LAYERS, N_KV, sum(-(-(n + 64 + 6 * t) // 16) for n in lengths) + 8, page_rows=16, device=DEV)
                       for _ in range(2))
    requests = [prompts(model, cache, lengths)[0] for cache in (eager, captured)]
    settings = [Settings(b), Settings(b)]
    tokens = torch.zeros((b, t), dtype=torch.long, device=DEV)
    table, eager_table = (torch.full((b, width), -1, dtype=torch.int32, device=DEV) for _ in range(2))
    lens, eager_lens, counts = (torch.zeros((b,), dtype=torch.int32, device=DEV) for _ in range(3))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):   # (no rows: nothing is written)
        step(model, captured, settings[1], tokens, table, lens, counts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        token, logprob = step(model, captured, settings[1], tokens, table, lens, counts)
    at = torch.arange(b, device=DEV)[:, None] * 17 + torch.arange(t, device=DEV)
    for i in range(6):
        news = [1 + (i + j) % t for j in range(b)]
        for s in settings:
            s.uniforms.copy_(torch.rand((b,), generator=torch.Generator().manual_seed(i)))
            s.options["temperature"].fill_(0.5 + 0.3 * i)
        if i == 3:   # the second request of the captured side ends up in other pages
            for cache, own in zip((eager, captured), requests):
                other = cache.fork(own[-1])
                cache.close(own[-1])
                own[-1] = other
            spare = captured.open()
            captured.reserve([spare], 33)
            captured.close(requests[1][0])
            requests[1][0] = captured.open()
            eager.close(requests[0][0])
            requests[0][0] = eager.open()
            captured.compact()
        for cache, own in zip((eager, captured), requests):
            cache.reserve(own, news)
        eager.batch(requests[0], news, table=eager_table, lens=eager_lens)
        captured.batch(requests[1], news, table=table, lens=lens)
        counts.copy_(torch.tensor(news, dtype=torch.int32))
        expect = step(model, eager, settings[0], at % VOCAB, eager_table, eager_lens, counts)
        tokens.copy_(at % VOCAB)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(token, expect[0]) and torch.equal(logprob, expect[1])
        for layer in range(LAYERS):
            for j, (x, y) in enumerate(zip(*requests)):
                a = kernels.paged_read(eager, layer, eager_table[j:j + 1], torch.zeros_like(eager_lens[:1]), 600, lens=eager_lens[j:j + 1])
                c = kernels.paged_read(captured, layer, table[j:j + 1], torch.zeros_like(lens[:1]), 600, lens=lens[j:j + 1])
                assert all(torch.equal(m, n) for m, n in zip(a, c))
        for cache, own in zip((eager, captured), requests):
            cache.advance(own, news)
        at = token.clamp(min=0)[:, None] + torch.arange(t, device=DEV)


@pytest.mark.parametrize("default", ["cpu", "cuda:0"])
def test_default_device_and_threads(gpu, default):
    """A default device changes nothing, and threads with streams and pools of their own
    do not meet (capacities on both sides of the one-launch rule)."""
    model, lengths = Model(), [1200, 30, 500]

    def answers():
        cache = PagedKVCache(LAYERS, N_KV, 64, page_rows=64, device=DEV)
        requests, token = prompts(model, cache, lengths)
        result = [token]
        for _ in range(3):
            cache.reserve(requests, 1)
            table, lens = cache.batch(requests, 1)
            token, logprob = step(model, cache, Settings(3), token.clamp(min=0)[:, None], table, lens)
            cache.advance(requests, 1)
            result += [token, logprob]
        one = cache.fork(requests[1])
        cache.reserve([one], 1)
        result += step(model, cache, Settings(1), result[-2][:1, None].clamp(min=0), *cache.batch([one], 1))
        return result

    want = answers()
    with torch.device(default):
        got = answers()
    assert all(torch.equal(x, y) for x, y in zip(want, got))
    torch.cuda.synchronize()

    def work(_):
        with torch.cuda.stream(torch.cuda.Stream()):
            results = [answers() for _ in range(3)]
            torch.cuda.current_stream().synchronize()
        return results

    with ThreadPoolExecutor(3) as pool:
        for results in pool.map(work, range(3)):
            for got in results:
                assert all(torch.equal(x, y) for x, y in zip(want, got))
