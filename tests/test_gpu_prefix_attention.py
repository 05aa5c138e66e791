"""Attention over a shared prefix (kernels.shared_prefix_attention) against the
definition in float64, value by value."""

from __future__ import annotations

import math

import pytest
import torch

from leanstack_amd import _lib, kernels
from leanstack_amd.kv_cache import ArenaKVCache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
D = 128
SCALE = D ** -0.5


def _normal(gen, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * std).bfloat16()


def _request(b, t, n_q, n_kv, prefix, rows, seed=0, std=1.5):
    """Inputs whose rows behind the written ones are NaN; lengths from 0 to all."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    q = _normal(gen, b, n_q, t, D, std=std)
    far = torch.full((2, n_kv, prefix + 40, D), math.nan, device=DEV, dtype=torch.bfloat16)
    far[:, :, :prefix] = _normal(gen, 2, n_kv, prefix, D)
    near = _normal(gen, 2, b, n_kv, rows, D)
    lens = torch.randint(0, rows + 1, (b,), generator=gen, device=DEV).int()
    lens[-1] = rows
    lens[b // 2] = min(t, rows)
    if b > 3:
        lens[1] = 0
    for i, n in enumerate(lens.tolist()):
        near[:, i, :, n:] = math.nan
    return q, far[0, :, :prefix], far[1, :, :prefix], near[0], near[1], lens


def _oracle(q, prefix_k, prefix_v, k, v, lens, scale):
    """float64 result [B, T, n_q * d] and a bound on the kernel's distance from it.

    A weight is off by its rounding to bf16, half a step, 2^-8 of it, and by its
    score's error: 128 fp32 additions, each one step, 2^-23, of the sum of
    magnitudes, and a few steps in the exponent (below 2^-16 together for
    exponents up to 2^6).  Normalised weights that are off by a share e move the
    result by at most e / (1 - e) of sum w |v - out|.  P V adds fp32 additions, one
    step of sum w |v| per row and per part; the output is rounded once, by 2^-8."""
    b, n_q, t, d = q.shape
    n_kv = prefix_k.shape[0]
    out = torch.zeros((b, t, n_q, d), device=DEV, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for i, length in enumerate(lens.tolist()):
        length = min(max(length, 0), k.shape[2])
        for j in range(t):
            own = max(0, length - (t - 1 - j))
            keys = torch.cat((prefix_k.double(), k[i, :, :own].double()), 1)
            values = torch.cat((prefix_v.double(), v[i, :, :own].double()), 1)
            n = keys.shape[1]
            if n == 0:
                continue
            heads = q[i, :, j].double().view(n_kv, n_q // n_kv, d)
            turned = keys.transpose(1, 2).contiguous()
            w = torch.softmax(torch.bmm(heads, turned) * scale, -1)
            size = torch.bmm(heads.abs(), turned.abs()).amax(-1, keepdim=True) * abs(scale)
            o = torch.bmm(w, values)
            e = 2.0 ** -8 + 2 * 128 * 2.0 ** -23 * size + 2.0 ** -16
            spread = torch.stack([(w[:, g, :, None] * (values - o[:, g, None]).abs()).sum(1) for g in range(w.shape[1])], 1)
            mass = torch.bmm(w, values.abs())
            err = e / (1 - e) * spread + (n + 80) * 2.0 ** -23 * mass
            out[i, j] = o.view(n_q, d)
            bound[i, j] = (err + (o.abs() + err) * 2.0 ** -8).view(n_q, d)
    return out.view(b, t, n_q * d), bound.view(b, t, n_q * d)


def _check(got, inputs, scale=SCALE):
    expect, bound = _oracle(*inputs, scale)
    assert got.shape == expect.shape and got.dtype == torch.bfloat16
    diff = (got.double() - expect).abs()
    over = diff - bound
    assert bool((over <= 0).all()), f"{float(over.max())} over the bound, {int((over > 0).sum())} values"


CASES = [
    # one launch: b, t, n_q, n_kv, prefix, rows
    (1, 1, 4, 1, 0, 1), (1, 1, 32, 8, 1, 0), (3, 1, 8, 8, 31, 33), (2, 5, 32, 8, 40, 64), (5, 1, 32, 4, 300, 200),
    (1, 40, 4, 4, 100, 60), (2, 16, 16, 2, 0, 500), (4, 2, 24, 8, 128, 129), (7, 1, 5, 5, 33, 31),
    # parts added up; few query rows
    (1, 1, 32, 8, 4097, 0), (2, 3, 32, 8, 1000, 300), (3, 1, 8, 1, 515, 1000), (16, 1, 4, 1, 700, 40), (1, 5, 32, 8, 0, 700),
    (4, 1, 48, 4, 600, 257),
    # 128 query rows to an item
    (40, 1, 32, 8, 600, 70), (9, 8, 32, 8, 1025, 130), (130, 1, 8, 8, 2000, 5), (5, 33, 12, 4, 515, 600),
    (33, 1, 16, 2, 513, 0), (20, 16, 4, 1, 0, 600), (65, 1, 3, 3, 511, 2),
    (70, 1, 32, 8, 1000, 70), (49, 1, 4, 1, 2000, 300), (200, 1, 8, 8, 1537, 0), (33, 7, 4, 4, 801, 40), (97, 2, 8, 4, 31, 900),
]


@pytest.mark.parametrize("case", CASES)
def test_prefix_attention(gpu, case):
    inputs = _request(*case, seed=sum(case))
    got = kernels.shared_prefix_attention(*inputs, SCALE)
    _check(got, inputs)
    assert torch.equal(got, kernels.shared_prefix_attention(*inputs, SCALE))


@pytest.mark.parametrize("case", [(2, 1, 32, 8, 16384, 300), (1, 4, 8, 2, 40000, 4096), (64, 1, 8, 2, 16384, 64)])
def test_long_contexts(gpu, case):
    inputs = _request(*case, seed=1)
    _check(kernels.shared_prefix_attention(*inputs, SCALE), inputs)


@pytest.mark.parametrize("case", [(3, 1, 8, 2, 64, 40), (3, 4, 8, 2, 64, 40), (3, 4, 8, 2, 900, 300), (40, 2, 8, 2, 900, 300)])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0, 1e-30])
def test_scales(gpu, case, scale):
    """Negative and zero scales, and scores up to several hundred."""
    inputs = _request(*case, seed=2, std=0.3 if scale == 3.0 else 1.5)
    _check(kernels.shared_prefix_attention(*inputs, scale), inputs, scale)


def test_rising_and_falling_scores(gpu):
    """Maxima that rise and fall by hundreds from step to step, and rows beside
    which all others vanish."""
    for case in ((2, 2, 4, 1, 300, 100), (2, 2, 4, 1, 2000, 300), (40, 2, 4, 1, 2000, 300)):
        q, pk, pv, k, v, lens = _request(*case, seed=3)
        for keys in (pk, k):
            n = keys.shape[-2]
            ramp = torch.linspace(-20, 20, n, device=DEV).view(n, 1)
            keys.copy_((keys.float() * 0.1 + ramp * torch.where(torch.arange(n, device=DEV) // 96 % 2 == 0, 1, -1).view(n, 1)).bfloat16())
        q.copy_((q.float() * 0.02 + 0.5).bfloat16())
        lens.fill_(k.shape[2])
        v.copy_(torch.nan_to_num(v))
        k.copy_(torch.nan_to_num(k))
        _check(kernels.shared_prefix_attention(q, pk, pv, k, v, lens, 1.0), (q, pk, pv, k, v, lens), 1.0)


@pytest.mark.parametrize("case", [(4, 1, 8, 2, 0, 64), (4, 3, 8, 2, 0, 64), (4, 3, 8, 2, 0, 700), (40, 3, 8, 2, 0, 700)])
def test_queries_that_see_no_row_give_zeros(gpu, case):
    inputs = _request(*case, seed=4)
    lens = inputs[-1]
    lens[:3] = torch.tensor([0, 1, -7], device=DEV, dtype=torch.int32)
    lens[3] = 2**31 - 1
    inputs[3][3], inputs[4][3] = 0.5, 0.25
    inputs[3][1, :, :1], inputs[4][1, :, :1] = 0.5, 0.25
    got = kernels.shared_prefix_attention(*inputs, SCALE)
    t = case[1]
    assert not bool(got[0].any()) and not bool(got[2].any()) and not bool(got[1, : t - 1].any())
    assert bool((got[1, t - 1] == 0.25).all()) and bool((got[3] == 0.25).all())
    far = _request(case[0], t, 8, 2, 0, 0)
    assert not bool(kernels.shared_prefix_attention(*far, SCALE).any())


@pytest.mark.parametrize("prefix,b", [(100, 2), (1000, 2), (1000, 40), (1000, 60)])
@pytest.mark.parametrize("t", [1, 6])
def test_infinities_and_nan(gpu, prefix, b, t):
    """Where they are seen they act as in torch's softmax and product; a query that
    does not see a row is not touched by it, in K or in V."""
    rows = 50
    q, pk, pv, k, v, lens = _request(b, t, 8, 2, prefix, rows, seed=5)
    lens[0] = 33
    k[0, :, :33], v[0, :, :33] = 0.25, torch.randn(33, D, device=DEV).bfloat16()
    q[0], pk[0, 3] = q[0].abs() + 0.1, -math.inf       # head 0: a row that weighs nothing for request 0
    base = kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE)
    assert bool(base[0].isfinite().all())
    if t > 1:
        # request 0's last two rows: seen by its last two queries (and one) alone
        k[0, 0, 31], v[0, 1, 31, 5], v[0, 1, 32, 6], k[0, 0, 32] = math.nan, math.inf, math.nan, math.inf
        got = kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE)
        rest = [i for i in range(b) if i != 0]
        assert torch.equal(got[rest].nan_to_num(7.0), base[rest].nan_to_num(7.0))
        assert torch.equal(got[0, : t - 2], base[0, : t - 2])
        heads, old = got[0].view(t, 8, D), base[0].view(t, 8, D)
        assert bool(heads[t - 2:, :4].isnan().all())
        assert bool((heads[t - 2:, 4:, 5] == math.inf).all()) and bool(heads[t - 1, 4:, 6].isnan().all())
        assert bool((heads[t - 2, 4:, 6].isfinite()).all())
        others = [i for i in range(D) if i not in (5, 6)]
        assert torch.equal(heads[t - 2:, 4:][..., others], old[t - 2:, 4:][..., others])
    # the prefix's last row: an infinity, and what fills the step up behind it
    pv[1, prefix - 1, 9], pk[1, prefix - 2, 0] = -math.inf, 0.0
    got = kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE).view(b, t, 8, D)
    assert bool((got[:, :, 4:, 9] == -math.inf).all())
    # every row -inf: NaN, as 0 / 0
    pk[:], k[:] = -math.inf, -math.inf
    q.copy_(q.abs() + 0.1)
    assert bool(kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE).isnan().all())


def test_last_own_row_infinite(gpu):
    """What stands for the rows past a request's last does not make a NaN of its infinity."""
    for case in ((3, 1, 8, 2, 64, 45), (3, 1, 8, 2, 900, 45), (40, 1, 8, 2, 900, 45), (50, 1, 8, 2, 900, 45)):
        q, pk, pv, k, v, lens = _request(*case, seed=6)
        lens.fill_(37)
        k[:, :, :37], v[:, :, :37] = 0.1, 0.5
        v[:, :, 36, 2] = math.inf
        got = kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE).view(case[0], 8, D)
        assert bool((got[..., 2] == math.inf).all())
        assert bool(got[..., [i for i in range(D) if i != 2]].isfinite().all())


@pytest.mark.parametrize("case", [(3, 2, 8, 2, 70, 50), (3, 2, 8, 2, 700, 300), (40, 1, 8, 2, 700, 300), (60, 1, 8, 2, 700, 300)])
def test_strides(gpu, case):
    """Caches with rows of all heads together, a layer of an ArenaKVCache, one
    request's rows for all, q before its transposition, a given output."""
    b, t, n_q, n_kv, prefix, rows = case
    q, pk, pv, k, v, lens = _request(*case, seed=7)
    expect = kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE)
    tk, tv = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
    fk, fv = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (pk, pv))
    assert tk.stride() != k.stride() and fk.stride() != pk.stride()
    assert torch.equal(kernels.shared_prefix_attention(q, fk, fv, tk, tv, lens, SCALE), expect)
    cache = ArenaKVCache(2, n_kv, D, prefix + 9, device=DEV)
    cache.write_rows(1, pk, pv)
    ck, cv = (x[0] for x in cache.attended(1))
    before = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    odd = torch.empty(q.numel() + 1, device=DEV, dtype=torch.bfloat16)[1:].view_as(q)
    odd.copy_(q)
    for form in (before, odd, q.repeat_interleave(2, 3)[..., ::2]):
        assert torch.equal(kernels.shared_prefix_attention(form, ck, cv, k, v, lens, SCALE), expect)
    room = torch.full((expect.numel() + 64,), 3.0, device=DEV).bfloat16()
    out = room[32:-32].view_as(expect)
    assert kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE, out=out) is out and torch.equal(out, expect)
    assert bool((room[:32] == 3).all()) and bool((room[-32:] == 3).all())
    lens.fill_(t)
    one_k, one_v = k[-1:].expand(b, -1, -1, -1), v[-1:].expand(b, -1, -1, -1)
    inputs = (q, pk, pv, one_k, one_v, lens)
    _check(kernels.shared_prefix_attention(*inputs, SCALE), inputs)


def test_offsets_past_32_bits(gpu):
    """Requests and heads more than 2^32 bytes apart."""
    b, n_kv, s = 3, 2, 40
    wide = torch.empty((b, n_kv, 6_000_000, D), device=DEV, dtype=torch.bfloat16)  # 1.5 GB per head
    q, pk, pv, k, v, lens = _request(b, 1, 8, n_kv, 600, s, seed=8)
    wide[:, :, -s:] = k
    far_v = torch.empty_like(wide)
    far_v[:, :, -s:] = v
    expect = kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE)
    got = kernels.shared_prefix_attention(q, pk, pv, wide[:, :, -s:], far_v[:, :, -s:], lens, SCALE)
    assert torch.equal(got, expect)
    wide[0, 0, 5_000_000:5_000_600] = pk[0]
    wide[0, 1, 5_000_000:5_000_600] = pk[1]
    far_v[0, 0, 5_000_000:5_000_600] = pv[0]
    far_v[0, 1, 5_000_000:5_000_600] = pv[1]
    far = wide[0, :, 5_000_000:5_000_600], far_v[0, :, 5_000_000:5_000_600]
    assert torch.equal(kernels.shared_prefix_attention(q, *far, k, v, lens, SCALE), expect)


def test_refuses_caches_it_cannot_read_in_place(gpu):
    q, pk, pv, k, v, lens = _request(3, 1, 8, 2, 70, 50, seed=7)
    odd = torch.zeros(pk.numel() + 1, device=DEV, dtype=torch.bfloat16)[1:].view(2, 70, D)
    with pytest.raises(ValueError, match="aligned"):
        kernels.shared_prefix_attention(q, odd, odd, k, v, lens, SCALE)
    with pytest.raises(ValueError, match="lens is on"):
        kernels.shared_prefix_attention(q, pk, pv, k, v, lens.cpu(), SCALE)
    with pytest.raises(ValueError, match="prefix_v is on"):
        kernels.shared_prefix_attention(q, pk.contiguous(), pv.contiguous().cpu(), k, v, lens, SCALE)


def test_empty_batch(gpu):
    empty = _request(2, 1, 8, 2, 64, 10)
    q, pk, pv, k, v, lens = empty
    assert kernels.shared_prefix_attention(q[:0], pk, pv, k[:0], v[:0], lens[:0], SCALE).shape == (0, 1, 8 * D)
    assert kernels.shared_prefix_attention(q[:, :, :0], pk, pv, k, v, lens, SCALE).shape == (2, 0, 8 * D)


@pytest.mark.parametrize("case", [(3, 1, 32, 8, 200, 100), (3, 4, 32, 8, 700, 300), (40, 1, 32, 8, 700, 300), (60, 1, 32, 8, 700, 300)])
def test_captured_and_on_two_streams(gpu, case):
    """Replays follow lens and the rows as they are then; a batch grows row by
    row; calls on two streams and two graphs share nothing."""
    b, t, n_q, n_kv, prefix, rows = case
    two = _lib.load().lsk_prefix_attention_workspace_bytes(b, t, n_q, n_kv, prefix, rows) > 0
    assert two == (prefix == 700)
    q, pk, pv, k, v, lens = _request(*case, seed=9)
    k.copy_(torch.nan_to_num(k, nan=0.3)), v.copy_(torch.nan_to_num(v, nan=0.2))
    kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE)))
    for step in range(4):
        lens.copy_((lens + 1).clamp(max=rows))
        q.copy_(q.flip(0))
        expect = kernels.shared_prefix_attention(q, pk, pv, k, v, lens, SCALE)
        for graph, out in graphs:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, expect)
    other = _request(*case, seed=10)
    pairs = [(q, pk, pv, k, v, lens), other]
    expect = [kernels.shared_prefix_attention(*p, SCALE) for p in pairs]
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(5):
        for stream, p in zip(streams, pairs):
            with torch.cuda.stream(stream):
                results.append(kernels.shared_prefix_attention(*p, SCALE))
    torch.cuda.synchronize()
    for i, out in enumerate(results):
        assert torch.equal(out, expect[i % 2])
