"""Decode and verify steps of a batch of requests that share a prompt, have
adapters of their own and constrained answers: the result of each such operator against
its definition on the inputs that it was really given, and captured steps against
eager ones."""

from __future__ import annotations

from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from leanstack_amd import _lib, kernels
from leanstack_amd.adapters import AdapterStore
from leanstack_amd.kv_cache import ArenaKVCache
from leanstack_amd.layout import PackedWeight
from tests import test_gpu_adapters as adapters_of
from tests import test_gpu_constrain as constraints_of
from tests import test_gpu_prefix_attention as attention_of
from tests.helpers import seeded_normal

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
H, N_Q, N_KV, D, INTER, VOCAB, LAYERS = 512, 8, 2, 128, 768, 2000, 2
EPS, SCALE = 1e-6, 128 ** -0.5
SHAPES = {"qkv": ((N_Q + 2 * N_KV) * D, H), "o": (H, N_Q * D), "gate_up": (2 * INTER, H), "down": (H, INTER)}
COUNT, RANK = 5, 16


class Model:
    """Random weights, adapters of every projection, a prompt's cache and tables."""

    def __init__(self, prefix):
        self.weights, self.adapters, self.stores = [], [], []
        for layer in range(LAYERS):
            w, lows, stores = {}, {}, {}
            for i, (name, (n, k)) in enumerate(SHAPES.items()):
                layout = _lib.LAYOUT_MFMA16X32_GATEUP if name == "gate_up" else _lib.LAYOUT_MFMA16X32
                w[name] = PackedWeight.from_rowmajor(seeded_normal((n, k), k ** -0.5, 40 * layer + i).to(DEV), layout)
                lows[name] = adapters_of._adapters(COUNT, n, k, [16, 3, 8, 16, 1], 1000 * layer + 100 * i)
                stores[name] = adapters_of._store(lows[name], n, k, RANK, gate_up=name == "gate_up")
            self.weights.append(w), self.adapters.append(lows), self.stores.append(stores)
        self.norm = (1 + seeded_normal((H,), 0.1, 7)).to(DEV)
        self.qk_norm = (1 + seeded_normal((D,), 0.1, 8)).to(DEV)
        self.embed = seeded_normal((VOCAB, H), 1.0, 9).to(DEV)
        self.head = PackedWeight.from_rowmajor(seeded_normal((VOCAB, H), 0.1, 10).to(DEV), _lib.LAYOUT_MFMA16X32)
        angle = torch.arange(4096)[:, None] * 1e4 ** (-torch.arange(D // 2) / (D // 2))
        self.cos, self.sin = angle.cos().bfloat16().to(DEV), angle.sin().bfloat16().to(DEV)
        self.prefix = prefix
        self.cache = ArenaKVCache(LAYERS, N_KV, D, prefix + 24, device=DEV)
        for layer in range(LAYERS):
            self.cache.write_rows(layer, seeded_normal((N_KV, prefix, D), 1.0, 50 + layer).to(DEV),
                                  seeded_normal((N_KV, prefix, D), 1.0, 60 + layer).to(DEV))


class Requests:
    """What a batch of b requests holds: tokens, lengths, own rows, settings."""

    def __init__(self, b, rows):
        gen = torch.Generator().manual_seed(3)
        self.k, self.v = (torch.full((LAYERS, b, N_KV, rows, D), float("nan"), dtype=torch.bfloat16, device=DEV)
                          for _ in range(2))
        self.lens = torch.randint(0, 4, (b,), generator=gen).int().to(DEV)
        for i, n in enumerate(self.lens.tolist()):
            self.k[:, i, :, :n], self.v[:, i, :, :n] = 0.3, 0.2
        self.index = (torch.arange(b) % (COUNT + 1) - 1).int().to(DEV)     # every adapter, and none
        self.history = torch.randint(0, VOCAB, (b, 64), generator=gen).int().to(DEV)
        self.history_lens = torch.full((b,), 9, dtype=torch.int32, device=DEV)
        self.prompt_lens = torch.full((b,), 5, dtype=torch.int32, device=DEV)
        self.repetition = (1 + torch.rand(b, generator=gen)).to(DEV)
        self.presence = torch.rand(b, generator=gen).to(DEV)
        self.bias_ids = torch.randint(0, VOCAB, (b, 7), generator=gen).int().to(DEV)
        self.bias_values = torch.randn(b, 7, generator=gen).to(DEV)
        self.allowed = torch.randint(-2**31, 2**31, (b, (VOCAB + 31) // 32), generator=gen, dtype=torch.int64).int().to(DEV)

    def parts(self):
        return [self.k, self.v, self.lens, self.history, self.history_lens]


def _step(model, req, tokens, seen=None):
    """Logits and greedy tokens behind `tokens` [B, T]; the last of them becomes part of
    the history.  seen: gets (operator, inputs, result) of every call."""
    b, t = tokens.shape
    note = seen.append if seen is not None else lambda _: None
    rows = torch.arange(b, device=DEV)[:, None]
    at = req.lens.long()[:, None] + torch.arange(t, device=DEV)
    cos, sin = model.cos[at + model.prefix], model.sin[at + model.prefix]
    index = req.index.repeat_interleave(t)
    req.lens.add_(t)
    hidden = model.embed[tokens]

    def project(layer, name, x, residual=None):
        silu = name == "gate_up"
        epilogue = _lib.EPI_SILU_MUL if silu else _lib.EPI_RESIDUAL_ADD if residual is not None else _lib.EPI_NONE
        weight, store = model.weights[layer][name], model.stores[layer][name]
        out = kernels.lora_linear(x, weight, store, index, epilogue=epilogue, residual=residual)
        note(("adapters", (layer, name, x, residual, index), out))
        return out

    for layer in range(LAYERS):
        normed = kernels.rmsnorm_rows(hidden, model.norm, EPS)
        qkv = project(layer, "qkv", normed)
        q, k = kernels.qk_norm_rope(qkv, model.qk_norm, model.qk_norm, EPS, cos, sin, num_attention_heads=N_Q,
                                    num_key_value_heads=N_KV)
        v = qkv[..., (N_Q + N_KV) * D:].view(b, t, N_KV, D)
        req.k[layer][rows, :, at], req.v[layer][rows, :, at] = k.transpose(1, 2), v
        pk, pv = (x[0] for x in model.cache.attended(layer))
        inputs = (q, pk, pv, req.k[layer], req.v[layer], req.lens)
        attended = kernels.shared_prefix_attention(*inputs, SCALE)
        note(("attention", tuple(x.clone() for x in inputs) if seen is not None else None, attended))
        hidden = project(layer, "o", attended, hidden)
        normed = kernels.rmsnorm_rows(hidden, model.norm, EPS)
        hidden = project(layer, "down", project(layer, "gate_up", normed), hidden)
    last = kernels.rmsnorm_rows(hidden[:, -1].contiguous(), model.norm, EPS)
    if b <= _lib.DECODE_MAX_M:
        logits = torch.empty((b, VOCAB), device=DEV)
        kernels.lm_head_argmax(last, model.head, logits_out=logits)
    else:
        logits = kernels.linear(last, model.head)
    settings = dict(history=req.history, history_lens=req.history_lens, prompt_lens=req.prompt_lens,
                    repetition=req.repetition, presence=req.presence, bias_ids=req.bias_ids,
                    bias_values=req.bias_values, allowed=req.allowed)
    values, token = kernels.constrain_logits(logits, **settings)
    note(("constraints", {k: x.clone() for k, x in settings.items()} | {"logits": logits} if seen is not None else None,
          (values, token)))
    req.history.scatter_(1, req.history_lens.long()[:, None], token.int()[:, None])
    req.history_lens.add_(1)
    return values, token


def _check(model, seen):
    for kind, inputs, result in seen:
        if kind == "attention":
            attention_of._check(result, inputs)
        elif kind == "adapters":
            layer, name, x, residual, index = inputs
            weight, lows = model.weights[layer][name], model.adapters[layer][name]
            gate_up = name == "gate_up"
            if gate_up:   # both halves in packed order
                order = torch.arange(2 * INTER).view(2, INTER // 16, 16).transpose(0, 1).reshape(-1)
                lows = [(a, low[order], s) for a, low, s in lows]
                weight = PackedWeight(weight.data, weight.n, weight.k, _lib.LAYOUT_MFMA16X32)
            epilogue = _lib.EPI_RESIDUAL_ADD if residual is not None else _lib.EPI_NONE
            y = kernels.linear(x, weight, epilogue=epilogue, residual=residual).flatten(0, 1)
            adapters_of._check(result.flatten(0, 1), y.cpu(), x.flatten(0, 1).cpu(), lows, index.cpu(), gate_up)
        else:
            z, bound = constraints_of._oracle(inputs.pop("logits").cpu(), **{k: x.cpu() for k, x in inputs.items()})
            constraints_of._check(result[0], result[1], z, bound)


@pytest.mark.parametrize("b,t,prefix", [(7, 1, 300), (12, 1, 1000), (16, 1, 40), (5, 4, 700), (60, 1, 1100), (33, 3, 900)])
def test_steps_against_the_definitions(gpu, b, t, prefix):
    model, req = Model(prefix), Requests(b, 40)
    tokens = torch.arange(b * t, device=DEV).view(b, t) * 31 % VOCAB
    for _ in range(3):
        seen = []
        _, token = _step(model, req, tokens, seen)
        _check(model, seen)
        assert len(seen) == LAYERS * 5 + 1
        # (a verify block's other tokens are drafts)
        tokens = torch.cat((token[:, None], (token[:, None] + torch.arange(1, t, device=DEV)) % VOCAB), 1)


@pytest.mark.parametrize("b,prefix", [(12, 300), (12, 1000), (60, 1100)])
def test_captured_steps_are_the_eager_ones(gpu, b, prefix):
    """One captured decode step, replayed: token by token what eager steps give, also
    after an adapter has been replaced between replays."""
    model = Model(prefix)
    eager, req = Requests(b, 40), Requests(b, 40)
    start = torch.arange(b, device=DEV)[:, None] * 17 % VOCAB
    tokens = start.clone()
    saved = [x.clone() for x in req.parts()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):   # (linear's workspace is allocated outside the capture)
        _step(model, req, tokens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        values, token = _step(model, req, tokens)
        tokens.copy_(token.clamp(min=0)[:, None])
    for x, old in zip(req.parts(), saved):
        x.copy_(old)
    tokens.copy_(start)
    at = start
    for step in range(5):
        if step == 3:
            a, low, s = adapters_of._adapters(1, *SHAPES["qkv"], [11], 77)[0]
            model.stores[0]["qkv"].load(2, a.to(DEV), low.to(DEV), s)
        expect, pick = _step(model, eager, at)
        at = pick.clamp(min=0)[:, None]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(values, expect) and torch.equal(token, pick) and torch.equal(tokens, at)
        for x, y in zip(req.parts(), eager.parts()):
            assert torch.equal(x.nan_to_num(7.0) if x.is_floating_point() else x,
                               y.nan_to_num(7.0) if y.is_floating_point() else y)


@pytest.mark.parametrize("default", ["cpu", "cuda:0"])
def test_default_device_and_threads(gpu, default):
    """A default device changes nothing, and threads with streams of their own do
    not meet."""
    model = Model(300)
    tokens = torch.arange(12, device=DEV)[:, None] * 17 % VOCAB
    values, token = _step(model, Requests(12, 40), tokens)
    req = Requests(12, 40)
    with torch.device(default):
        store = AdapterStore(COUNT, *SHAPES["o"], RANK, device=DEV)
        for slot, (a, b, s) in enumerate(model.adapters[0]["o"]):
            store.load(slot, a, b, s)
        assert torch.equal(store.a_tiles, model.stores[0]["o"].a_tiles)
        assert torch.equal(store.b_tiles, model.stores[0]["o"].b_tiles)
        got = _step(model, req, tokens)
    assert torch.equal(got[0], values) and torch.equal(got[1], token)
    torch.cuda.synchronize()

    def work(_):
        with torch.cuda.stream(torch.cuda.Stream()):
            results = [_step(model, Requests(12, 40), tokens) for _ in range(4)]
            torch.cuda.current_stream().synchronize()
        return results

    with ThreadPoolExecutor(3) as pool:
        for results in pool.map(work, range(3)):
            assert all(torch.equal(v, values) and torch.equal(t, token) for v, t in results)
