"""Operators of a batch of requests on one resident model, as cases that can be timed and checked.

Between the projections that all requests share, a batched decode or verify step has three parts of its own:

  prefix_attention  attention of every request's new tokens over a prefix that all of them share (a system prompt,
                    a document) and over the rows that each request has cached since
  adapters          the low-rank adapters that the requests chose, added to a shared projection's rows
  constraints       penalties for repeated tokens, biases and grammar masks on the logits, and the greedy token

Sizes are the Qwen3-4B geometry's where a case does not say otherwise.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

from leanstack_amd.geometry import QWEN3_4B as G

own = False

DEV = "cuda"
D = G.head_dim
H, I, V = G.hidden_size, G.intermediate_size, G.vocab_size
NQ, NKV = G.num_attention_heads, G.num_key_value_heads
SHAPES = {"qkv": (G.qkv_dim, H), "o": (H, G.q_dim), "gate_up": (2 * I, H), "down": (H, I)}  # (N, K)


def listed() -> list[dict]:
    return [
        # a verify block of four drafted tokens of one request, over its short context
        {"name": "attend_verify_1x5", "op": "prefix_attention", "b": 1, "t": 5, "n_q": NQ, "n_kv": NKV, "prefix": 300,
         "own_min": 5, "own_max": 40, "own_rows": 64},
        # a small batch over a prompt bucket, answers of different length, one slot empty
        {"name": "attend_12", "op": "prefix_attention", "b": 12, "t": 1, "n_q": NQ, "n_kv": NKV, "prefix": 1024,
         "own_min": 0, "own_max": 333, "own_rows": 512},
        # a full batch over a long document, long answers
        {"name": "attend_64", "op": "prefix_attention", "b": 64, "t": 1, "n_q": NQ, "n_kv": NKV, "prefix": 8191,
         "own_min": 1, "own_max": 1000, "own_rows": 1088},
        # many verify blocks over the longest context that the caches hold
        {"name": "attend_verify_48x4", "op": "prefix_attention", "b": 48, "t": 4, "n_q": NQ, "n_kv": NKV, "prefix": 16000,
         "own_min": 4, "own_max": 300, "own_rows": 320},
        # one token of one request, a small adapter
        {"name": "adapters_o_1", "op": "adapters", "proj": "o", "m": 1, "adapters": 4, "rank": 8, "plain_rows": 0, "runs": 1},
        # a decode batch, every row with an adapter of its own choice
        {"name": "adapters_qkv_16", "op": "adapters", "proj": "qkv", "m": 16, "adapters": 24, "rank": 16, "plain_rows": 3,
         "runs": 1},
        # a larger batch with larger adapters on the longest input rows
        {"name": "adapters_down_64", "op": "adapters", "proj": "down", "m": 64, "adapters": 32, "rank": 64, "plain_rows": 9,
         "runs": 1},
        # prompts of several requests in one call, the MLP's first projection with its SiLU(gate) * up
        {"name": "adapters_gate_up_2000", "op": "adapters", "proj": "gate_up", "m": 2000, "adapters": 8, "rank": 32,
         "plain_rows": 300, "runs": 250},
        # one request: repeated tokens of a short answer
        {"name": "constrain_1", "op": "constraints", "m": 1, "v": V, "dtype": "float32", "history": 600, "bias": 0,
         "mask": False, "penalties": True},
        # a verify block under a grammar only
        {"name": "constrain_mask_5", "op": "constraints", "m": 5, "v": V, "dtype": "float32", "history": 0, "bias": 0,
         "mask": True, "penalties": False},
        # a vocabulary of odd size in bf16, everything on
        {"name": "constrain_bf16_37", "op": "constraints", "m": 37, "v": 50257, "dtype": "bfloat16", "history": 2000,
         "bias": 40, "mask": True, "penalties": True},
        # a full batch late in a long context, everything on
        {"name": "constrain_128", "op": "constraints", "m": 128, "v": V, "dtype": "float32", "history": 8000, "bias": 300,
         "mask": True, "penalties": True},
    ]


def _spread(rng, low: int, high: int) -> int:
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _costs_no_more(case: dict) -> bool:
    w, of_op = work(case), [work(c) for c in listed() if c["op"] == case["op"]]
    return all(w[key] <= max(o[key] for o in of_op) for key in ("bytes", "flops"))


def draw(rng) -> dict:
    op = rng.choice(("prefix_attention", "adapters", "constraints"))
    while True:
        if op == "prefix_attention":
            n_q, n_kv = rng.choice(((NQ, NKV), (NQ, NKV), (NQ, NKV), (8, 1), (16, 16), (32, 4), (8, 4)))
            t = rng.choice((1, 1, 1, 2, 3, 5, 8, 16))
            rows = _spread(rng, t, 2048)
            case = {"op": op, "b": _spread(rng, 1, 96), "t": t, "n_q": n_q, "n_kv": n_kv,
                    "prefix": _spread(rng, 1, 16384) - (1 if rng.random() < 0.3 else 0), "own_min": rng.randint(0, t),
                    "own_max": rng.randint(t, rows), "own_rows": rows}
        elif op == "adapters":
            m = _spread(rng, 1, 4096)
            runs = _spread(rng, 1, m) if m > 64 else 1
            case = {"op": op, "proj": rng.choice(tuple(SHAPES)), "m": m, "adapters": _spread(rng, 1, 48),
                    "rank": rng.choice((4, 8, 16, 16, 24, 32, 64, 100, 128)), "plain_rows": rng.randint(0, m // 2),
                    "runs": runs}
        else:
            penalties, mask = rng.choice(((True, True), (True, True), (True, False), (False, True)))
            case = {"op": op, "m": _spread(rng, 1, 160), "v": rng.choice((V, V, V // 8, 32000, 50257, 128256, 1003)),
                    "dtype": rng.choice(("float32", "float32", "bfloat16")),
                    "history": _spread(rng, 1, 16384) if penalties else 0, "bias": rng.choice((0, 0, 7, 300)), "mask": mask,
                    "penalties": penalties}
        if _costs_no_more(case):
            return case


def _own_lens(case) -> list[int]:
    """Rows that each request has cached: even steps over the case's range."""
    b, low, high = case["b"], case["own_min"], case["own_max"]
    return [high] if b == 1 else [low + (high - low) * i // (b - 1) for i in range(b)]


def work(case) -> dict:
    if case["op"] == "prefix_attention":
        b, t, n_q, n_kv, prefix = (case[key] for key in ("b", "t", "n_q", "n_kv", "prefix"))
        lens = _own_lens(case)
        seen = sum(prefix + max(0, n - (t - 1 - i)) for n in lens for i in range(t))
        return {"bytes": (prefix + sum(lens)) * n_kv * D * 2 * 2 + b * t * n_q * D * 2 * 2 + 4 * b,
                "flops": 4 * D * n_q * seen}
    if case["op"] == "adapters":
        n, k = SHAPES[case["proj"]]
        m, r = case["m"], case["rank"]
        rows = m - case["plain_rows"]
        used = min(case["adapters"], -(-rows // case["runs"]))
        n_out = n // 2 if case["proj"] == "gate_up" else n
        return {"bytes": 2 * (rows * k + m * n + m * n_out + used * r * (n + k)) + 4 * m + 4 * used,
                "flops": 2 * rows * r * (n + k)}
    m, v = case["m"], case["v"]
    item = 4 if case["dtype"] == "float32" else 2
    return {"bytes": m * (2 * v * item + 4 * case["history"] + 8 * case["bias"] + (v // 8 if case["mask"] else 0) + 28),
            "flops": m * v * (4 if case["penalties"] else 1)}


# ------------------------------------------------------------------ inputs


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(gen, shape, std=1.0, mean=0.0, dtype=torch.bfloat16):
    return torch.empty(shape, device=DEV, dtype=torch.float32).normal_(mean, std, generator=gen).to(dtype)


def _shuffled(gen, values, dtype=torch.int32):
    values = torch.tensor(values, device=DEV, dtype=dtype)
    return values[torch.randperm(values.numel(), generator=gen, device=DEV)]


def _prefix_attention_inputs(case, gen) -> SimpleNamespace:
    b, t, n_q, n_kv, prefix, rows = (case[key] for key in ("b", "t", "n_q", "n_kv", "prefix", "own_rows"))
    # scores of a standard deviation near 2, as normed and rotated heads give
    s = SimpleNamespace(q=_normal(gen, (b, n_q, t, D), 2.0), scale=D ** -0.5)
    # the prefix is the written part of a longer cache
    cache = _normal(gen, (2, n_kv, prefix + 64, D))
    s.prefix_k, s.prefix_v = cache[0, :, :prefix], cache[1, :, :prefix]
    s.k, s.v = _normal(gen, (b, n_kv, rows, D)), _normal(gen, (b, n_kv, rows, D))
    s.lens = _shuffled(gen, _own_lens(case))
    return s


def _adapters_inputs(case, gen) -> SimpleNamespace:
    n, k = SHAPES[case["proj"]]
    m, r, count = case["m"], case["rank"], case["adapters"]
    s = SimpleNamespace(silu=case["proj"] == "gate_up")
    s.x, s.y = _normal(gen, (m, k)), _normal(gen, (m, n))  # for gate_up: 16 gate columns, their 16 up columns, ...
    s.a, s.b = _normal(gen, (count, r, k), k ** -0.5), _normal(gen, (count, n, r), 0.05)
    s.scale = torch.rand((count,), generator=gen, device=DEV) * 1.5 + 0.5
    rows = m - case["plain_rows"]
    # consecutive rows of one request share its adapter; rows of requests without one come last
    chosen = torch.arange(rows, device=DEV) // case["runs"]
    names = torch.randperm(count, generator=gen, device=DEV)
    index = torch.cat((names[chosen % count], torch.full((m - rows,), -1, device=DEV, dtype=torch.long)))
    if case["runs"] == 1:  # a decode batch: in the order in which the requests came
        index = index[torch.randperm(m, generator=gen, device=DEV)]
    s.index = index.to(torch.int32)
    if own:  # the store that a server keeps its adapters in
        from leanstack_amd.adapters import AdapterStore
        s.store = AdapterStore.of(s.a, s.b, s.scale, gate_up=s.silu)
    return s


def _constraints_inputs(case, gen) -> SimpleNamespace:
    m, v, length = case["m"], case["v"], case["history"]
    dtype = torch.float32 if case["dtype"] == "float32" else torch.bfloat16
    s = SimpleNamespace(logits=_normal(gen, (m, v), 3.0, dtype=dtype), history=None, history_lens=None, prompt_lens=None,
                        repetition=None, frequency=None, presence=None, bias_ids=None, bias_values=None, allowed=None)
    if case["penalties"]:
        # token frequencies fall off as in text; contexts of half to full length, a third of them the prompt
        rank = torch.rand((m, length), generator=gen, device=DEV, dtype=torch.float64)
        names = torch.randperm(v, generator=gen, device=DEV)
        s.history = names[(torch.exp(rank * math.log(v)).long() - 1).clamp(0, v - 1)].to(torch.int32)
        s.history_lens = _shuffled(gen, [length - (length // 2) * i // m for i in range(m)])
        s.prompt_lens = s.history_lens // 3
        s.repetition = torch.rand((m,), generator=gen, device=DEV) * 0.5 + 1.0
        s.frequency = torch.rand((m,), generator=gen, device=DEV) * 0.5
        s.presence = torch.rand((m,), generator=gen, device=DEV) * 0.5
    if case["bias"]:
        s.bias_ids = torch.rand((m, v), generator=gen, device=DEV).topk(case["bias"]).indices.to(torch.int32)
        s.bias_values = _normal(gen, (m, case["bias"]), 4.0, dtype=torch.float32)
    if case["mask"]:
        # a grammar allows a quarter of the vocabulary's words, or nearly all of it
        words = torch.randint(0, 1 << 32, (3, m, -(-v // 32)), generator=gen, device=DEV)
        few, most = words[0] & words[1], words[0] | words[1] | words[2]
        loose = (torch.arange(m, device=DEV) % 3 == 2)[:, None]
        bits = torch.where(loose, most, few)
        s.allowed = (bits - ((bits >> 31) << 32)).to(torch.int32)  # bit 31 is an int32's sign
    return s


_INPUTS = {"prefix_attention": _prefix_attention_inputs, "adapters": _adapters_inputs, "constraints": _constraints_inputs}


def prepare(case, seed) -> SimpleNamespace:
    state = _INPUTS[case["op"]](case, _generator(seed))
    state.op = case["op"]
    return state


# ------------------------------------------------------------------ one pass


def _bits(allowed, v):
    """[M, V] truth values of the words."""
    at = torch.arange(v, device=allowed.device)
    return ((allowed[:, at // 32] >> (at % 32)) & 1).bool()


def _visible(s, rows):
    """[B, 1, T, 1, rows]: whether query t of a request sees a row that the request cached."""
    t = s.q.shape[2]
    n = s.lens.long()[:, None] - torch.arange(t - 1, -1, -1, device=s.lens.device)
    return (torch.arange(rows, device=s.lens.device) < n[..., None])[:, None, :, None]


def _attend(s, dtype):
    """Both parts' scores under one softmax; [B, T, n_q * d] in `dtype`."""
    b, n_q, t, d = s.q.shape
    n_kv, prefix, rows = s.prefix_k.shape[0], s.prefix_k.shape[1], s.k.shape[2]
    g = n_q // n_kv
    q = s.q.to(dtype).view(b, n_kv, g, t, d).transpose(2, 3).contiguous()  # [B, n_kv, T, G, d]
    q_all = q.transpose(0, 1).reshape(n_kv, b * t * g, d)
    far = torch.matmul(q_all, s.prefix_k.to(dtype).transpose(1, 2).contiguous()) * s.scale
    far = far.view(n_kv, b, t, g, prefix).transpose(0, 1)
    near = torch.matmul(q.view(b, n_kv, t * g, d), s.k.to(dtype).transpose(2, 3).contiguous()) * s.scale
    near = near.view(b, n_kv, t, g, rows).masked_fill(~_visible(s, rows), -math.inf)
    top = near.amax(-1, keepdim=True)
    top = torch.maximum(top, far.amax(-1, keepdim=True)) if prefix else top
    top = top.clamp(min=torch.finfo(dtype).min)
    far, near = torch.exp(far - top), torch.exp(near - top)
    total = far.sum(-1, keepdim=True) + near.sum(-1, keepdim=True)
    out = torch.matmul(far.transpose(0, 1).reshape(n_kv, b * t * g, prefix), s.prefix_v.to(dtype).contiguous())
    out = out.view(n_kv, b, t, g, d).transpose(0, 1)
    out = out + torch.matmul(near.view(b, n_kv, t * g, rows), s.v.to(dtype)).view(b, n_kv, t, g, d)
    out = torch.where(total > 0, out / total, 0)
    return out.permute(0, 2, 1, 3, 4).reshape(b, t, n_q * d)


def _adapt(s, dtype):
    """Every row through every adapter, the others' columns zero in between."""
    count, r, k = s.a.shape
    m, n = s.y.shape
    hidden = torch.matmul(s.x.to(dtype), s.a.to(dtype).view(count * r, k).t().contiguous()).view(m, count, r)
    chosen = s.index[:, None] == torch.arange(count, device=s.index.device)
    hidden = torch.where(chosen[..., None], hidden * s.scale.to(dtype)[:, None], 0)
    z = s.y.to(dtype) + torch.matmul(hidden.view(m, count * r),
                                     _columns(s.b.to(dtype), s.silu).transpose(1, 2).reshape(count * r, n))
    if not s.silu:
        return z
    z = z.view(m, n // 32, 2, 16)
    gate, up = z[:, :, 0], z[:, :, 1]
    return (gate / (1 + torch.exp(-gate)) * up).reshape(m, n // 2)


def _columns(b, silu):
    """Rows of b ([gate; up] for gate_up) in the order of y's columns."""
    if not silu:
        return b
    count, n, r = b.shape
    return b.view(count, 2, n // 32, 16, r).transpose(1, 2).reshape(count, n, r)


def _constrain(s, dtype):
    """The logits under the request's penalties, biases and mask, in `dtype`."""
    z = s.logits.to(dtype)
    m, v = z.shape
    if s.history is not None:
        at = torch.arange(s.history.shape[1], device=z.device)
        written = at < s.history_lens[:, None]
        answer = written & (at >= s.prompt_lens[:, None])
        seen = torch.zeros((m, v), device=z.device, dtype=torch.int32)
        count = torch.zeros((m, v), device=z.device, dtype=torch.int32)
        seen.scatter_add_(1, s.history.long(), written.int())
        count.scatter_add_(1, s.history.long(), answer.int())
        rho = s.repetition.to(dtype)[:, None]
        z = torch.where(seen > 0, torch.where(z > 0, z / rho, z * rho), z)
        less = z - s.frequency.to(dtype)[:, None] * count - s.presence.to(dtype)[:, None]
        z = torch.where(count > 0, less, z)
    if s.bias_ids is not None:
        z = z + torch.zeros_like(z).scatter_(1, s.bias_ids.long(), s.bias_values.to(dtype))
    if s.allowed is not None:
        z = z.masked_fill(~_bits(s.allowed, v), -math.inf)
    return z


def _greedy(logits):
    top, token = logits.max(-1)  # the lowest index of equal values, chosen below
    at = torch.arange(logits.shape[1], device=logits.device)
    token = torch.where(logits == top[:, None], at, logits.shape[1]).amin(-1)
    return torch.where(top > -math.inf, token, -1)


def run(state):
    s = state
    if own:
        from leanstack_amd import _lib, kernels
        if s.op == "prefix_attention":
            return kernels.shared_prefix_attention(s.q, s.prefix_k, s.prefix_v, s.k, s.v, s.lens, s.scale)
        if s.op == "adapters":
            return kernels.lora_add(s.y, s.x, s.store, s.index,
                                    epilogue=_lib.EPI_SILU_MUL if s.silu else _lib.EPI_NONE)
        return kernels.constrain_logits(
            s.logits, history=s.history, history_lens=s.history_lens, prompt_lens=s.prompt_lens, repetition=s.repetition,
            frequency=s.frequency, presence=s.presence, bias_ids=s.bias_ids, bias_values=s.bias_values, allowed=s.allowed)
    if s.op == "prefix_attention":
        return _attend(s, torch.float32).to(torch.bfloat16)
    if s.op == "adapters":
        return _adapt(s, torch.float32).to(torch.bfloat16)
    logits = _constrain(s, torch.float32).to(s.logits.dtype)
    return logits, _greedy(logits)


# ------------------------------------------------------------------ in 64 bits, request by request


def _exact_attention(s):
    b, n_q, t, d = s.q.shape
    n_kv = s.prefix_k.shape[0]
    out = torch.zeros((b, t, n_q, d), device=DEV, dtype=torch.float64)
    far_k, far_v = s.prefix_k.double(), s.prefix_v.double()
    for i, length in enumerate(s.lens.tolist()):
        keys = torch.cat((far_k, s.k[i, :, :length].double()), 1)
        values = torch.cat((far_v, s.v[i, :, :length].double()), 1)
        for j in range(t):
            n = far_k.shape[1] + max(0, length - (t - 1 - j))
            if n:
                q = s.q[i, :, j].double().view(n_kv, n_q // n_kv, d)
                weights = torch.softmax(torch.bmm(q, keys[:, :n].transpose(1, 2).contiguous()) * s.scale, -1)
                out[i, j] = torch.bmm(weights, values[:, :n].contiguous()).view(n_q, d)
    return out.view(b, t, n_q * d)


def _exact_adapters(s):
    z = s.y.double()
    half = z.shape[1] // 2
    block = torch.arange(half, device=DEV)
    gate = block // 16 * 32 + block % 16  # where y holds gate and up of an output
    for i in range(s.a.shape[0]):
        rows = (s.index == i).nonzero().view(-1)
        delta = s.x[rows].double() @ s.a[i].double().t() @ s.b[i].double().t() * s.scale[i].double()
        if s.silu:
            z[rows[:, None], gate] += delta[:, :half]
            z[rows[:, None], gate + 16] += delta[:, half:]
        else:
            z[rows] += delta
    return torch.sigmoid(z[:, gate]) * z[:, gate] * z[:, gate + 16] if s.silu else z


def _exact_constraints(s):
    z = s.logits.double()
    m, v = z.shape
    for i in range(m):
        row = z[i]
        if s.history is not None:
            past = s.history[i, : int(s.history_lens[i])].long()
            seen = past.unique()
            rho = float(s.repetition[i])
            row[seen] = torch.where(row[seen] > 0, row[seen] / rho, row[seen] * rho)
            tokens, count = past[int(s.prompt_lens[i]):].unique(return_counts=True)
            row[tokens] -= float(s.frequency[i]) * count + float(s.presence[i])
        if s.bias_ids is not None:
            row[s.bias_ids[i].long()] += s.bias_values[i].double()
        if s.allowed is not None:
            words = s.allowed[i].view(torch.uint8).view(-1, 1)  # little-endian bytes, 8 tokens each
            open_ = (words >> torch.arange(8, device=DEV, dtype=torch.uint8)) & 1
            row[open_.reshape(-1)[:v] == 0] = -math.inf
    rounded = z.to(s.logits.dtype).cpu().double().numpy()
    tokens = [int(r.argmax()) if r.max() > -math.inf else -1 for r in rounded]
    return z, torch.tensor(tokens, device=DEV)


_EXACT = {"prefix_attention": _exact_attention, "adapters": _exact_adapters, "constraints": _exact_constraints}


def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))
