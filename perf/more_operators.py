"""Operators of a server that keeps many requests' keys and values in 8 bits, in pages, as cases that can be timed and checked.

A batched step appends its new rows to the cache, attends over it and draws its tokens; between steps pages move:

  rows       new key and value rows rounded to 8 bits and stored, and the rows that the cache then stands for read back
             (as a request that moves to a contiguous cache, or a test of the rounding, takes them)
  attention  of every request's new tokens over its pages: single tokens, verify blocks, prompts in chunks
  pages      pages copied in all layers: a request that forks, a pool that is compacted
  sampling   a token from every row of logits: temperature, top-k, min-p and top-p, from given random numbers

The cache: pages of rows per kv head; 16 rows of a head are a block of 2048 bytes (e4m3) with one exponent byte, a
value being its byte's times 2 ^ (exponent - 127).  Sizes are the Qwen3-4B geometry's where a case does not say otherwise.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import torch

from leanstack_amd.geometry import QWEN3_4B as G

own = False

DEV = "cuda"
D = G.head_dim
V = G.vocab_size
NQ, NKV, LAYERS = G.num_attention_heads, G.num_key_value_heads, G.num_hidden_layers
BLOCK = 16  # rows that share an exponent
LEAST, MOST = -100, 119  # exponents


def listed() -> list[dict]:
    return [
        # one request's new token
        {"name": "rows_1", "op": "rows", "b": 1, "t": 1, "n_kv": NKV, "page": 64, "min": 777, "max": 777, "ragged": False},
        # a decode batch, contexts of any length
        {"name": "rows_96x1", "op": "rows", "b": 96, "t": 1, "n_kv": NKV, "page": 64, "min": 1, "max": 4000, "ragged": False},
        # prompts of several requests, the shorter ones padded, the first chunk or a later one
        {"name": "rows_prompts_3x1999", "op": "rows", "b": 3, "t": 1999, "n_kv": NKV, "page": 64, "min": 1999, "max": 5003,
         "ragged": True},
        # one request's token over a short context
        {"name": "attend_1", "op": "attention", "b": 1, "t": 1, "n_q": NQ, "n_kv": NKV, "page": 64, "min": 900, "max": 900,
         "ragged": False},
        # a full decode batch: contexts from a greeting to a long document
        {"name": "attend_64", "op": "attention", "b": 64, "t": 1, "n_q": NQ, "n_kv": NKV, "page": 64, "min": 17, "max": 8001,
         "ragged": False},
        # verify blocks of up to four drafted tokens
        {"name": "attend_verify_24x5", "op": "attention", "b": 24, "t": 5, "n_q": NQ, "n_kv": NKV, "page": 32, "min": 5,
         "max": 3001, "ragged": True},
        # chunks of two long prompts behind what is already cached of them
        {"name": "attend_prompts_2x1500", "op": "attention", "b": 2, "t": 1500, "n_q": NQ, "n_kv": NKV, "page": 64, "min": 4000,
         "max": 7001, "ragged": False},
        # a request forks into several: the last page of each, in every layer
        {"name": "fork_3", "op": "pages", "layers": LAYERS, "n_kv": NKV, "page": 64, "pages": 24, "moved": 3},
        # a pool is compacted after its batch has shrunk
        {"name": "compact_50", "op": "pages", "layers": LAYERS, "n_kv": NKV, "page": 64, "pages": 120, "moved": 50},
        # one request's token, the usual filters
        {"name": "sample_1", "op": "sampling", "m": 1, "v": V, "dtype": "float32", "top_k": 50, "top_p": True, "min_p": False,
         "greedy": 0},
        # a vocabulary of odd size in bf16 (many equal logits), drawn by min-p alone
        {"name": "sample_bf16_37", "op": "sampling", "m": 37, "v": 50257, "dtype": "bfloat16", "top_k": 0, "top_p": False,
         "min_p": True, "greedy": 0},
        # a full batch, everything on, some requests greedy
        {"name": "sample_128", "op": "sampling", "m": 128, "v": V, "dtype": "float32", "top_k": 1000, "top_p": True,
         "min_p": True, "greedy": 5},
    ]


def _spread(rng, low: int, high: int) -> int:
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _costs_no_more(case: dict) -> bool:
    w, of_op = work(case), [work(c) for c in listed() if c["op"] == case["op"]]
    return all(w[key] <= max(o[key] for o in of_op) for key in ("bytes", "flops"))


def draw(rng) -> dict:
    op = rng.choice(("rows", "attention", "attention", "pages", "sampling", "sampling"))
    while True:
        if op == "rows":
            t = rng.choice((1, 1, 2, 5, 16, 33, _spread(rng, 64, 4096)))
            most = _spread(rng, max(t, 2), 8192)
            case = {"op": op, "b": _spread(rng, 1, 160), "t": t, "n_kv": rng.choice((NKV, NKV, 1, 4, 16)),
                    "page": rng.choice((16, 32, 64, 64, 128)), "min": rng.randint(1, most), "max": most,
                    "ragged": rng.random() < 0.4}
        elif op == "attention":
            n_q, n_kv = rng.choice(((NQ, NKV), (NQ, NKV), (NQ, NKV), (8, 1), (16, 16), (32, 4), (8, 4), (40, 8)))
            t = rng.choice((1, 1, 1, 1, 2, 3, 5, 8, 16, _spread(rng, 17, 2048)))
            most = _spread(rng, max(t, 2), 16384)
            case = {"op": op, "b": _spread(rng, 1, 128), "t": t, "n_q": n_q, "n_kv": n_kv,
                    "page": rng.choice((16, 32, 64, 64, 128)), "min": rng.randint(1, most), "max": most,
                    "ragged": rng.random() < 0.4}
        elif op == "pages":
            pages = _spread(rng, 8, 240)
            case = {"op": op, "layers": rng.choice((LAYERS, 12, 5)), "n_kv": rng.choice((NKV, 1, 4)),
                    "page": rng.choice((16, 32, 64, 128)), "pages": pages, "moved": _spread(rng, 1, pages // 2)}
        else:
            m = _spread(rng, 1, 160)
            case = {"op": op, "m": m, "v": rng.choice((V, V, V // 8, 32000, 50257, 128256, 1003)),
                    "dtype": rng.choice(("float32", "float32", "bfloat16")), "top_k": rng.choice((0, 1, 20, 50, 1000)),
                    "top_p": rng.random() < 0.6, "min_p": rng.random() < 0.4, "greedy": rng.choice((0, 0, m // 3))}
        if _costs_no_more(case):
            return case


def _steps(case) -> list[int]:
    """Rows that each request has cached, the new ones among them: even steps over the case's range."""
    b, low, high = case["b"], case["min"], case["max"]
    return [high] if b == 1 else [low + (high - low) * i // (b - 1) for i in range(b)]


def _new(case) -> list[int]:
    """How many of its t new rows each request has."""
    lens, t = _steps(case), case["t"]
    return [min(n, t - (i * 5 % t if case["ragged"] else 0)) for i, n in enumerate(lens)]


def work(case) -> dict:
    if case["op"] == "rows":
        values = sum(_new(case)) * case["n_kv"] * D * 2  # of k and of v
        old = sum((n - new) % BLOCK for n, new in zip(_steps(case), _new(case))) * case["n_kv"] * D * 2
        # new rows in, the begun blocks in; bytes stored and read back, the values out
        return {"bytes": 2 * values + 3 * old + 2 * values + 2 * (values + old), "flops": 4 * values}
    if case["op"] == "attention":
        lens, new, n_q, n_kv = _steps(case), _new(case), case["n_q"], case["n_kv"]
        seen = sum(c * n - c * (c - 1) // 2 for n, c in zip(lens, new))
        return {"bytes": sum(lens) * n_kv * D * 2 + sum(-(-n // BLOCK) for n in lens) * n_kv * 2
                + (sum(new) + case["b"] * case["t"]) * n_q * D * 2 + 8 * case["b"], "flops": 4 * D * n_q * seen}
    if case["op"] == "pages":
        page = case["layers"] * 2 * case["n_kv"] * (case["page"] * D + case["page"] // BLOCK)
        return {"bytes": 2 * case["moved"] * page, "flops": 0}
    m, v = case["m"], case["v"]
    return {"bytes": m * (v * (4 if case["dtype"] == "float32" else 2) + 32), "flops": 16 * m * v}


# ------------------------------------------------------------------ the cache's format


def _power(e):
    """2 ^ e, as float32."""
    return ((e + 127) << 23).view(torch.float32)


def _exponent(x):
    """Per block [..., BLOCK, D] of float32: the least e with |x| <= 448 * 2 ^ e, of the finite values."""
    top = torch.where(torch.isfinite(x), x, 0).abs().amax((-2, -1))
    part, e = torch.frexp(top)  # part in [1/2, 1)
    e = torch.where(part <= 0.875, e - 9, e - 8)
    return torch.where(top > 0, e, LEAST).clamp(LEAST, MOST).to(torch.int32)


def _bytes_of(x, e):
    """float32 [..., BLOCK, D] in units of 2 ^ e, e [...], as bytes."""
    x = x * _power(-e)[..., None, None]
    fine = torch.isfinite(x)
    q = torch.where(fine, x, 0).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.where(fine, q, 0x7F)


def _values_of(q, e):
    return q.view(torch.float8_e4m3fn).to(torch.float32) * _power(e)[..., None, None]


def _pack(q):
    """Bytes [..., 2 (k, v), BLOCK, D] as blocks [..., 2, 2048]: the order in which a wave's lanes multiply them."""
    lead = q.shape[:-3]
    k = q[..., 0, :, :].reshape(*lead, BLOCK, 2, 4, 16)  # row, half, quarter of it, dim
    v = q[..., 1, :, :].reshape(*lead, 4, 4, 4, 2, 16)  # row / 4, row % 4, dim / 32, dim / 16 % 2, dim % 16
    n = len(lead)
    k = k.permute(*range(n), n + 1, n + 2, n, n + 3).reshape(*lead, 2048)
    v = v.permute(*range(n), n + 3, n, n + 4, n + 2, n + 1).reshape(*lead, 2048)
    return torch.stack((k, v), -2)


def _unpack(blocks):
    """Blocks [..., 2 (k, v), 2048] as bytes [..., 2, BLOCK, D]."""
    lead = blocks.shape[:-2]
    n = len(lead)
    k = blocks[..., 0, :].reshape(*lead, 2, 4, BLOCK, 16).permute(*range(n), n + 2, n, n + 1, n + 3)
    v = blocks[..., 1, :].reshape(*lead, 2, 4, 16, 4, 4).permute(*range(n), n + 1, n + 4, n + 3, n, n + 2)
    return torch.stack((k.reshape(*lead, BLOCK, D), v.reshape(*lead, BLOCK, D)), -3)


def _gathered(s, first, count):
    """Blocks first .. first + count - 1 (first [B]) of every request: bytes [B, count, n_kv, 2, BLOCK, D], exponents
    [B, count, n_kv, 2], and whether they are in the pool, [B, count]."""
    per_page = s.page // BLOCK
    block = first[:, None] + torch.arange(count, device=first.device)
    page = s.table.long().gather(1, (block // per_page).clamp(0, s.table.shape[1] - 1))
    there = (page >= 0) & (page < s.storage.shape[2]) & (block < s.table.shape[1] * per_page)
    page = torch.where(there, page, 0)
    at = block % per_page
    blocks = s.storage[s.layer].permute(1, 3, 2, 0, 4)[page, at]  # [B, count, n_kv, 2, 2048]
    e = s.scales[s.layer].permute(1, 3, 2, 0)[page, at].int() - 127
    return _unpack(blocks), e, there, page, at


# ------------------------------------------------------------------ inputs


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(gen, shape, std=1.0, dtype=torch.bfloat16):
    return torch.empty(shape, device=DEV, dtype=torch.float32).normal_(0.0, std, generator=gen).to(dtype)


def _pool(s, gen, layers, n_kv, pages, page):
    """A pool in use: values of a standard deviation that differs from block to block."""
    spread = torch.rand((layers, pages, n_kv, page // BLOCK, 2, 1, 1), generator=gen, device=DEV) * 1.5 + 0.5
    x = _normal(gen, (layers, pages, n_kv, page // BLOCK, 2, BLOCK, D), dtype=torch.float32) * spread
    e = _exponent(x)
    blocks = _pack(_bytes_of(x, e))
    s.storage = blocks.permute(0, 4, 1, 2, 3, 5).contiguous()  # [layers, 2, pages, n_kv, blocks, 2048]
    s.scales = (e + 127).to(torch.uint8).permute(0, 4, 1, 2, 3).contiguous()  # [layers, 2, pages, n_kv, blocks]
    s.page = page
    if own:  # the handle that a server keeps its pool in
        from leanstack_amd.paged_cache import PagedKVCache
        s.cache = PagedKVCache.of(s.storage, s.scales)


def _requests(s, case, gen):
    """lens, counts and the page table of the case's requests: pages in any order, -1 behind the last."""
    lens, new = _steps(case), _new(case)
    need = [-(-n // case["page"]) for n in lens]
    pages = sum(need) + 3
    s.layer = 1
    _pool(s, gen, 2, case["n_kv"], pages, case["page"])
    order = torch.randperm(case["b"], generator=gen, device=DEV)
    names = torch.randperm(pages, generator=gen, device=DEV)
    need = torch.tensor(need, device=DEV)
    at = torch.arange(int(need.max()) + 1, device=DEV)
    first = need.cumsum(0) - need
    table = torch.where(at < need[:, None], names[(first[:, None] + at).clamp(max=pages - 1)], -1)
    s.table = table[order].to(torch.int32).contiguous()
    s.lens = torch.tensor(lens, device=DEV, dtype=torch.int32)[order]
    s.counts = torch.tensor(new, device=DEV, dtype=torch.int32)[order]
    # a batch that is not padded names no counts
    s.given = s.counts if new != [case["t"]] * case["b"] else None


def _rows_inputs(case, gen) -> SimpleNamespace:
    s = SimpleNamespace(t=case["t"])
    _requests(s, case, gen)
    b, t, n_kv = case["b"], case["t"], case["n_kv"]
    s.k = _normal(gen, (b, n_kv, t, D), 1.5)
    # values as they lie in the projection's rows, behind the query and key heads
    s.v = _normal(gen, (b, t, 3 * n_kv, D), 0.7)[:, :, 2 * n_kv:].transpose(1, 2)
    # what is read back: every block that the new rows touch
    s.starts = ((s.lens - s.counts) // BLOCK * BLOCK).to(torch.int32)
    s.rows = (t + 2 * BLOCK - 2) // BLOCK * BLOCK
    return s


def _attention_inputs(case, gen) -> SimpleNamespace:
    s = SimpleNamespace(scale=D ** -0.5)
    _requests(s, case, gen)
    # scores of a standard deviation near 2, as normed and rotated heads give
    s.q = _normal(gen, (case["b"], case["n_q"], case["t"], D), 1.6)
    return s


def _pages_inputs(case, gen) -> SimpleNamespace:
    s = SimpleNamespace()
    _pool(s, gen, case["layers"], case["n_kv"], case["pages"], case["page"])
    names = torch.randperm(case["pages"], generator=gen, device=DEV).to(torch.int32)
    s.src, s.dst = names[:case["moved"]].contiguous(), names[case["moved"]:2 * case["moved"]].contiguous()
    return s


def _sampling_inputs(case, gen) -> SimpleNamespace:
    m, v = case["m"], case["v"]
    dtype = torch.float32 if case["dtype"] == "float32" else torch.bfloat16
    # a few tokens stand out, as a language model's do
    logits = _normal(gen, (m, v), 2.5, dtype=torch.float32)
    s = SimpleNamespace(top_k=None, top_p=None, min_p=None)
    s.logits = (logits + 0.25 * logits.clamp(min=0).square()).to(dtype)

    def per_row(low, high):
        return torch.rand((m,), generator=gen, device=DEV) * (high - low) + low

    s.uniforms, s.temperature = per_row(0.0, 1.0), per_row(0.6, 1.3)
    s.temperature[:case["greedy"]] = 0.0
    if case["top_k"]:
        s.top_k = (per_row(0.5, 1.5) * case["top_k"]).int().clamp(min=1)
    if case["top_p"]:
        s.top_p = per_row(0.7, 1.0)
    if case["min_p"]:
        s.min_p = per_row(0.001, 0.1)
    return s


_INPUTS = {"rows": _rows_inputs, "attention": _attention_inputs, "pages": _pages_inputs, "sampling": _sampling_inputs}


def prepare(case, seed) -> SimpleNamespace:
    state = _INPUTS[case["op"]](case, _generator(seed))
    state.op = case["op"]
    return state


# ------------------------------------------------------------------ one pass


def _store(s):
    """The new rows in the pool: begun blocks with the larger of their exponent and the new rows'."""
    first = (s.lens - s.counts).clamp(min=0).long() // BLOCK
    count = s.rows // BLOCK
    q, e_old, there, page, at = _gathered(s, first, count)
    row = (first[:, None] + torch.arange(count, device=first.device))[..., None] * BLOCK + torch.arange(BLOCK, device=first.device)
    start = (s.lens - s.counts).long()[:, None, None]
    new = (row >= start) & (row < s.lens.long()[:, None, None]) & there[..., None]  # [B, count, BLOCK]
    old = (row < start)
    begun = old[..., 0] & new.any(-1)
    token = (row - start).clamp(0, s.t - 1).reshape(len(first), -1)
    b = torch.arange(len(first), device=first.device)[:, None]
    x = torch.stack((s.k.transpose(1, 2)[b, token], s.v.transpose(1, 2)[b, token]), 3).float()  # [B, rows, n_kv, 2, D]
    x = x.view(len(first), count, BLOCK, *x.shape[2:]).permute(0, 1, 3, 4, 2, 5)
    new = new[:, :, None, None, :, None]
    x = torch.where(new, x, 0)
    e = _exponent(x)
    e = torch.where(begun[..., None, None], torch.maximum(e, e_old), e)
    moved = _bytes_of(_values_of(q, e_old), e)
    q = torch.where(new, _bytes_of(x, e), torch.where((old & begun[..., None])[:, :, None, None, :, None], moved, q))
    touched = new.flatten(2).any(-1).nonzero(as_tuple=True)
    where = (slice(None), page[touched], slice(None), at[touched])
    s.storage[s.layer][where] = _pack(q)[touched].transpose(1, 2)
    s.scales[s.layer][where] = (e + 127).to(torch.uint8)[touched].transpose(1, 2)


def _read(s):
    """k and v [B, n_kv, rows, D] from `starts` on; zeros behind the last row."""
    q, e, there, _, _ = _gathered(s, s.starts.long() // BLOCK, s.rows // BLOCK)
    x = _values_of(q, e).permute(3, 0, 2, 1, 4, 5).flatten(3, 4)  # [2, B, n_kv, rows, D]
    row = s.starts.long()[:, None] + torch.arange(s.rows, device=q.device)
    fine = (row < s.lens[:, None]) & there.repeat_interleave(BLOCK, 1)
    x = torch.where(fine[:, None, :, None], x, 0).to(torch.bfloat16)
    return x[0], x[1]


def _attend(s):
    b, n_q, t, d = s.q.shape
    blocks = s.table.shape[1] * (s.page // BLOCK)
    q, e, there, _, _ = _gathered(s, torch.zeros_like(s.lens).long(), blocks)
    x = _values_of(q, e).permute(3, 0, 2, 1, 4, 5).flatten(3, 4)  # [2, B, n_kv, S, D]
    k, v = x[0], x[1]
    n_kv, rows = k.shape[1:3]
    at = torch.arange(t, device=q.device)
    seen = s.lens.long()[:, None] - (s.counts[:, None] - 1 - at)  # [B, T] rows that a query sees
    seen = torch.where(at < s.counts[:, None], seen, 0)
    fine = (torch.arange(rows, device=q.device) < seen[..., None]) & there.repeat_interleave(BLOCK, 1)[:, None]
    fine = fine[:, None, :, None]  # [B, 1, T, 1, S]
    groups = s.q.float().view(b, n_kv, n_q // n_kv, t, d).transpose(2, 3).reshape(b, n_kv, -1, d)
    w = torch.matmul(groups, k.transpose(2, 3).contiguous()).view(b, n_kv, t, n_q // n_kv, rows) * s.scale
    w = w.masked_fill(~fine, -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w.view(b, n_kv, -1, rows), v.contiguous()).view(b, n_kv, t, n_q // n_kv, d)
    out = torch.where(total > 0, out / total, 0)
    return out.permute(0, 2, 1, 3, 4).reshape(b, t, n_q * d).to(torch.bfloat16)


def _sample(s):
    """In whole multiples of 2 ^ -44 of the largest weight, so that no order of sums moves a border."""
    unit = float(1 << 44)
    x = s.logits.double()
    v = x.shape[1]
    top = x.amax(-1, keepdim=True)
    w = torch.where(x == top, 0.0, (x - top) / s.temperature.double()[:, None])
    w = torch.round(torch.exp(w) * unit).long()
    order = torch.argsort(x, dim=-1, descending=True, stable=True)
    w = w.gather(1, order)
    at = torch.arange(v, device=x.device)
    keep = (at == 0) | (s.temperature > 0)[:, None]
    if s.top_k is not None:
        keep &= at < s.top_k[:, None]
    if s.min_p is not None:
        keep &= w.double() >= s.min_p.double()[:, None] * unit
    w = torch.where(keep, w, 0)
    if s.top_p is not None:
        before = w.cumsum(-1) - w
        w = torch.where(before.double() < s.top_p.double()[:, None] * w.sum(-1, keepdim=True).double(), w, 0)
    kept = torch.zeros_like(w).scatter_(1, order, w)
    total = kept.sum(-1)
    target = (s.uniforms.double() * total.double()).floor().long()
    token = (kept.cumsum(-1) <= target[:, None]).sum(-1)
    return token, torch.log(kept.gather(1, token[:, None])[:, 0].double() / total.double()).float()


def run(state):
    s = state
    if own:
        from leanstack_amd import kernels
        if s.op == "rows":
            kernels.paged_append(s.cache, s.layer, s.k, s.v, s.table, s.lens, counts=s.given)
            return kernels.paged_read(s.cache, s.layer, s.table, s.starts, s.rows, lens=s.lens)
        if s.op == "attention":
            return kernels.paged_attention(s.q, s.cache, s.layer, s.table, s.lens, s.scale, counts=s.given)
        if s.op == "pages":
            kernels.copy_pages(s.cache, s.src, s.dst)
            return s.storage, s.scales
        return kernels.sample_logits(s.logits, s.uniforms, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p,
                                     min_p=s.min_p)
    if s.op == "rows":
        _store(s)
        return _read(s)
    if s.op == "attention":
        return _attend(s)
    if s.op == "pages":
        s.storage[:, :, s.dst.long()] = s.storage[:, :, s.src.long()]
        s.scales[:, :, s.dst.long()] = s.scales[:, :, s.src.long()]
        return s.storage, s.scales
    return _sample(s)


# ------------------------------------------------------------------ in 64 bits, request by request


def _stored(s, b, rows):
    """The first `rows` rows of request b as the pool's bytes stand for them, float64 [2 (k, v), n_kv, rows, D]: every byte
    by the format's place and its sign, exponent and fraction bits."""
    t, d = torch.arange(rows, device=DEV)[:, None], torch.arange(D, device=DEV)
    page, at = s.table[b].long()[t // s.page], t % s.page
    block, t = at // BLOCK, at % BLOCK
    place = torch.stack((d // 64 * 1024 + (d // 16 % 4 * 16 + t) * 16 + d % 16,
                         d // 16 % 2 * 1024 + (t // 4 * 16 + d % 16) * 16 + d // 32 * 4 + t % 4))  # [2, rows, D]
    kv, head = torch.arange(2, device=DEV)[:, None, None, None], torch.arange(s.storage.shape[3], device=DEV)[:, None, None]
    byte = s.storage[s.layer][kv, page[None], head, block[None], place[:, None]].int()
    e = s.scales[s.layer][kv, page[None], head, block[None]].double() - 127
    sign, power, fraction = byte >> 7, byte >> 3 & 15, byte & 7
    size = torch.where(power > 0, (8 + fraction).double() * torch.exp2(power.double() - 10), fraction.double() * 2.0 ** -9)
    return torch.where(sign > 0, -size, size) * torch.exp2(e)


def _nearest(x, e):
    """Multiples of the e4m3 step at x / 2 ^ e, ties to even, times 2 ^ e."""
    y = (x / 2.0 ** e).clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * 2.0 ** e


def _exact_rows(s):
    b, n_kv = s.k.shape[:2]
    out = torch.zeros((2, b, n_kv, s.rows, D), device=DEV, dtype=torch.float64)
    for i in range(b):
        n, new, first = int(s.lens[i]), int(s.counts[i]), int(s.starts[i])
        rows = torch.zeros((2, n_kv, s.rows, D), device=DEV, dtype=torch.float64)
        begun = n - new - first
        if begun:
            page, block = int(s.table[i, first // s.page]), first % s.page // BLOCK
            rows[:, :, :begun] = _stored(s, i, first + begun)[:, :, first:]
            was = s.scales[s.layer, :, page, :, block].double() - 127
        fresh = torch.stack((s.k[i, :, :new], s.v[i, :, :new])).double()
        rows[:, :, begun:begun + new] = fresh
        blocks = rows.view(2, n_kv, -1, BLOCK, D)
        mine = torch.zeros_like(rows)
        mine[:, :, begun:begun + new] = fresh
        top = mine.view_as(blocks).abs().amax((-2, -1))
        e = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** LEAST))).clamp(LEAST, MOST)
        if begun:
            e[:, :, 0] = torch.maximum(e[:, :, 0], was)
        out[:, i] = _nearest(blocks, e[..., None, None]).view_as(rows)
    return out[0], out[1]


def _exact_attention(s):
    b, n_q, t, d = s.q.shape
    n_kv = s.storage.shape[3]
    out = torch.zeros((b, t, n_q, d), device=DEV, dtype=torch.float64)
    for i in range(b):
        n, new = int(s.lens[i]), int(s.counts[i])
        keys, values = _stored(s, i, n)
        seen = n - new + 1 + torch.arange(new, device=DEV)
        hidden = torch.arange(n, device=DEV) >= seen[:, None]
        for j in range(n_kv):
            heads = slice(j * n_q // n_kv, (j + 1) * n_q // n_kv)
            scores = torch.matmul(s.q[i, heads, :new].double(), keys[j].t().contiguous()) * s.scale
            out[i, :new, heads] = torch.matmul(torch.softmax(scores.masked_fill(hidden, -math.inf), -1), values[j]).transpose(0, 1)
    return out.view(b, t, n_q * d)


def _exact_sampling(s):
    x = s.logits.double().cpu().numpy()
    tokens, logs = [], []
    for i, row in enumerate(x):
        ranked = np.lexsort((np.arange(len(row)), -row))
        temperature = float(s.temperature[i])
        if temperature <= 0:
            tokens.append(int(ranked[0]))
            logs.append(0.0)
            continue
        weight = np.rint(np.ldexp(np.exp((row - row.max()) / temperature), 44)).astype(np.int64)
        if s.top_k is not None:
            ranked = ranked[:int(s.top_k[i])]
        if s.min_p is not None:
            ranked = ranked[weight[ranked] >= float(s.min_p[i]) * 2.0 ** 44]
        if s.top_p is not None:
            sums = np.cumsum(weight[ranked])
            ranked = ranked[:1 + int(np.searchsorted(sums.astype(np.float64), float(s.top_p[i]) * float(sums[-1]), "left"))]
        ranked.sort()
        sums = np.cumsum(weight[ranked])
        token = ranked[np.searchsorted(sums, int(float(s.uniforms[i]) * float(sums[-1])), "right")]
        tokens.append(int(token))
        logs.append(math.log(int(weight[token]) / int(sums[-1])))
    return torch.tensor(tokens, device=DEV), torch.tensor(logs, device=DEV, dtype=torch.float64)


def exact(case, seed):
    if case["op"] == "pages":
        return None  # bytes moved: nothing is computed
    return {"rows": _exact_rows, "attention": _exact_attention, "sampling": _exact_sampling}[case["op"]](prepare(case, seed))
