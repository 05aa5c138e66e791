"""Low-rank adapters (kernels.lora_add, kernels.lora_linear) against the
definition in float64, value by value."""

from __future__ import annotations

import math

import pytest
import torch

from leanstack_amd import _lib, kernels
from leanstack_amd.adapters import AdapterStore
from leanstack_amd.layout import PackedWeight
from tests.helpers import seeded_normal

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
SILU = _lib.EPI_SILU_MUL


def _adapters(count, n, k, ranks, seed):
    """(A, B, scale) per adapter, on the CPU."""
    return [(seeded_normal((r, k), k ** -0.5, seed + 3 * i), seeded_normal((n, r), 0.1, seed + 3 * i + 1), 0.5 + 0.25 * i)
            for i, r in zip(range(count), ranks)]


def _store(adapters, n, k, rank, gate_up=False):
    store = AdapterStore(len(adapters), n, k, rank, gate_up=gate_up, device=DEV)
    for slot, (a, b, s) in enumerate(adapters):
        store.load(slot, a.to(DEV), b.to(DEV), s)
    return store


def _oracle(y, x, adapters, index, gate_up=False):
    """float64 result and a bound on the kernel's distance from it.

    h's K products and z's R are summed in fp32: at most one fp32 step, 2^-23, of
    the sum of magnitudes per addition; h's two bf16 parts lose 2^-17 of it; z is
    rounded once, by half a bf16 step, 2^-8 of it."""
    z = y.double().clone()
    err = torch.zeros_like(z)
    for m, i in enumerate(index.tolist()):
        if 0 <= i < len(adapters):
            a, b, s = adapters[i]
            z[m] += s * (b.double() @ (a.double() @ x[m].double()))
            size = s * (b.double().abs() @ (a.double().abs() @ x[m].double().abs()))
            err[m] = size * ((x.shape[1] + 2 * a.shape[0] + 8) * 2.0 ** -23 + 2.0 ** -16) + z[m].abs() * 2.0 ** -23
    if not gate_up:
        return z, err + (z.abs() + err) * 2.0 ** -8
    half = z.shape[1] // 2
    block = torch.arange(half)
    gate = block // 16 * 32 + block % 16
    g, u, dg, du = z[:, gate], z[:, gate + 16], err[:, gate], err[:, gate + 16]
    silu = g * torch.sigmoid(g)
    # |silu'| <= 1.1; the sigmoid on the hardware exp2 and reciprocal keeps 2^-17
    err = 1.1 * dg * (u.abs() + du) + silu.abs() * du + (silu * u).abs() * 2.0 ** -16
    return silu * u, err + ((silu * u).abs() + err) * 2.0 ** -8


def _check(got, y, x, adapters, index, gate_up=False):
    z, bound = _oracle(y, x, adapters, index, gate_up)
    got = got.cpu().double()
    assert got.shape == z.shape
    diff = (got - z).abs()
    assert bool((diff <= bound).all()), f"{float((diff - bound).max())} over the bound"


def _index(m, count, seed):
    """Adapters in any order, rows without one among them."""
    return torch.randint(-1, count, (m,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


@pytest.mark.parametrize("m,n,k,count,rank", [
    (1, 16, 32, 1, 1), (1, 2560, 4096, 4, 8), (2, 48, 64, 2, 16), (5, 80, 96, 3, 17), (15, 112, 288, 16, 5),
    (16, 6144, 2560, 20, 16), (17, 2560, 9728, 3, 64), (33, 512, 2048, 33, 100), (64, 2560, 9728, 9, 128),
    (130, 256, 512, 5, 48), (301, 1040, 2560, 4, 32), (40, 2560, 4096, 1, 96), (16, 32, 4096, 40, 128),
    (128, 528, 512, 60, 16), (129, 16, 32, 64, 3), (640, 2560, 4096, 9, 16), (200, 304, 9728, 3, 128), (1000, 96, 1024, 2, 64),
])
def test_lora_add(gpu, m, n, k, count, rank):
    adapters = _adapters(count, n, k, [max(1, rank - 3 * (i % 4)) for i in range(count)], seed=m)
    y, x = seeded_normal((m, n), 1.0, 1), seeded_normal((m, k), 1.0, 2)
    index = _index(m, count, m)
    store = _store(adapters, n, k, rank)
    dy, dx, di = y.to(DEV), x.to(DEV), index.to(DEV)
    got = kernels.lora_add(dy, dx, store, di)
    _check(got, y, x, adapters, index)
    assert torch.equal(got, kernels.lora_add(dy, dx, store, di))
    assert torch.equal(got.cpu()[index < 0], y[index < 0])
    assert torch.equal(dy.cpu(), y)
    assert kernels.lora_add(dy, dx, store, di, out=dy) is dy and torch.equal(dy, got)


@pytest.mark.parametrize("m,n,k,count,rank", [
    (1, 32, 32, 1, 4), (7, 192, 2560, 7, 16), (16, 19456, 2560, 3, 32), (50, 1024, 9728, 16, 128), (200, 320, 512, 2, 64),
    (300, 96, 2560, 5, 128), (129, 19456, 1024, 3, 16), (90, 160, 9728, 4, 48),
])
def test_lora_silu_mul(gpu, m, n, k, count, rank):
    adapters = _adapters(count, n, k, [rank] * count, seed=m)
    y, x = seeded_normal((m, n), 2.0, 1), seeded_normal((m, k), 1.0, 2)
    index = _index(m, count, m + 1)
    # the store takes [gate; up] rows; y's columns and the oracle's are in packed order
    rows = torch.arange(n).view(2, n // 32, 16).transpose(0, 1).reshape(-1)
    store = _store(adapters, n, k, rank, gate_up=True)
    got = kernels.lora_add(y.to(DEV), x.to(DEV), store, index.to(DEV), epilogue=SILU)
    _check(got, y, x, [(a, b[rows], s) for a, b, s in adapters], index, gate_up=True)


@pytest.mark.parametrize("k,rank", [(512, 16), (9728, 64)])  # one launch and two
@pytest.mark.parametrize("m", [16, 37, 150])
def test_rows_and_adapters_do_not_touch_each_other(gpu, m, k, rank):
    """A NaN or infinity in one row's x or y, or in an adapter, reaches only the
    rows that it is a part of; indices that name no adapter leave y; unused
    slots may hold anything."""
    n, count = 320, 6
    two = _lib.load().lsk_lora_workspace_bytes(m, n, k, rank // 16, count, 0) > 0
    assert two == (k == 9728 or m > 128)
    adapters = _adapters(count, n, k, [rank, rank - 1, rank, 3, rank, rank], seed=5)
    y, x = seeded_normal((m, n), 1.0, 1), seeded_normal((m, k), 1.0, 2)
    index = torch.arange(m, dtype=torch.int32) % 4
    index[5], index[6], index[9], index[10] = -1, count, 2**31 - 1, -2**31
    clean = _store(adapters, n, k, rank)
    expect = kernels.lora_add(y.to(DEV), x.to(DEV), clean, index.to(DEV)).cpu()
    _check(expect, y, x, adapters, index)
    adapters[4][0][:] = math.nan
    adapters[5][1][:] = math.inf
    adapters[2][1][7, 0] = math.inf    # adapter 2, column 7
    store = _store(adapters, n, k, rank)
    x[0, 11] = math.nan                # row 0 (adapter 0)
    x[3, 12] = math.inf                # row 3 (adapter 3, of a lower rank than the store's)
    y[1, 13] = math.nan
    x[5], x[6] = math.nan, math.inf    # rows without an adapter
    got = kernels.lora_add(y.to(DEV), x.to(DEV), store, index.to(DEV)).cpu()
    assert bool(got[0].isnan().all())
    z = y[3].double() + adapters[3][2] * (adapters[3][1].double() @ (adapters[3][0].double() @ x[3].double()))
    assert torch.equal(got[3].isnan(), z.isnan()) and torch.equal(got[3].isinf(), z.isinf())
    assert bool(got[1, 13].isnan())
    two_rows = index == 2
    assert not bool(got[two_rows, 7].isfinite().any())
    keep = torch.ones((m, n), dtype=torch.bool)
    keep[0], keep[3], keep[1, 13], keep[two_rows, 7] = False, False, False, False
    assert torch.equal(got[keep], expect[keep])
    assert torch.equal(got[5], y[5]) and torch.equal(got[6], y[6])


@pytest.mark.parametrize("runs", [1, 3, 50, 64, 100])
def test_prompts_of_several_requests(gpu, runs):
    """Consecutive rows of a request, adapters that change inside a tile of rows
    and at its edges, requests without one between them."""
    m, n, k, count = 333, 320, 512, 7
    adapters = _adapters(count, n, k, [16, 9, 30, 32, 1, 17, 32], seed=2)
    y, x = seeded_normal((m, n), 1.0, 1), seeded_normal((m, k), 1.0, 2)
    index = ((torch.arange(m) // runs) % (count + 1) - 1).int()
    got = kernels.lora_add(y.to(DEV), x.to(DEV), _store(adapters, n, k, 32), index.to(DEV))
    _check(got, y, x, adapters, index)
    rows = torch.arange(n).view(2, n // 32, 16).transpose(0, 1).reshape(-1)
    got = kernels.lora_add(y.to(DEV), x.to(DEV), _store(adapters, n, k, 32, gate_up=True), index.to(DEV), epilogue=SILU)
    _check(got, y, x, [(a, b[rows], s) for a, b, s in adapters], index, gate_up=True)


@pytest.mark.parametrize("m", [21, 140])
def test_strides_shapes_and_empty_calls(gpu, m):
    n, k = 96, 256
    adapters = _adapters(3, n, k, [9, 16, 4], seed=1)
    store = _store(adapters, n, k, 16)
    y, x, index = seeded_normal((m, n), 1.0, 1), seeded_normal((m, k), 1.0, 2), _index(m, 3, 4)
    dy, dx, di = y.to(DEV), x.to(DEV), index.to(DEV)
    expect = kernels.lora_add(dy, dx, store, di)
    wide_y, wide_x = torch.full((m, n + 24), 9.0, device=DEV).bfloat16(), torch.full((m, k + 40), 9.0, device=DEV).bfloat16()
    wide_y[:, 8:8 + n], wide_x[:, 16:16 + k] = dy, dx
    for fy, fx in ((wide_y[:, 8:8 + n], wide_x[:, 16:16 + k]), (dy.t().contiguous().t(), dx.repeat_interleave(2, 1)[:, ::2]),
                   (wide_y.clone()[:, 8:8 + n], dx.view(-1, 7, k)), (dy.view(1, m, n), dx.view(1, m, k))):
        assert torch.equal(kernels.lora_add(fy, fx, store, di).view(m, n), expect)
    shifted = torch.empty(m * k + 1, device=DEV, dtype=torch.bfloat16)[1:].view(m, k)
    shifted.copy_(dx)
    room = torch.full((m * n + 64,), 5.0, device=DEV).bfloat16()
    out = room[32:32 + m * n].view(m, n)
    assert kernels.lora_add(dy, shifted, store, di, out=out) is out and torch.equal(out, expect)
    assert bool((room[:32] == 5).all()) and bool((room[32 + m * n:] == 5).all())
    assert kernels.lora_add(dy[:0], dx[:0], store, di[:0]).shape == (0, n)
    one = kernels.lora_add(dy[4], dx[4], store, di[4:5])
    assert one.shape == (n,) and torch.equal(one, kernels.lora_add(dy[4:5], dx[4:5], store, di[4:5])[0])


def test_slots_are_loaded_replaced_and_cleared(gpu):
    n, k = 64, 128
    adapters = _adapters(4, n, k, [16, 7, 30, 1], seed=9)
    y, x = seeded_normal((4, n), 1.0, 1), seeded_normal((4, k), 1.0, 2)
    store = AdapterStore(3, n, k, 30, device=DEV)
    index = torch.tensor([0, 1, 2, 1], dtype=torch.int32)
    dy, dx, di = y.to(DEV), x.to(DEV), index.to(DEV)
    assert torch.equal(kernels.lora_add(dy, dx, store, di), dy)  # empty slots add nothing
    for slot in range(3):
        store.load(slot, adapters[slot][0].to(DEV), adapters[slot][1].to(DEV), adapters[slot][2])
    _check(kernels.lora_add(dy, dx, store, di), y, x, adapters[:3], index)
    store.load(2, adapters[3][0].to(DEV), adapters[3][1].to(DEV), adapters[3][2])  # rank 1 after rank 30
    now = [adapters[0], adapters[1], adapters[3]]
    _check(kernels.lora_add(dy, dx, store, di), y, x, now, index)
    store.load(1, torch.full_like(adapters[1][0], math.inf).to(DEV), adapters[1][1].to(DEV) * math.inf, 1.0)
    store.clear(1)
    _check(kernels.lora_add(dy, dx, store, di), y, x, [now[0], (now[1][0] * 0, now[1][1] * 0, 1.0), now[2]], index)
    again = AdapterStore.of(torch.stack([a[0] for a in _adapters(3, n, k, [5] * 3, 2)]).to(DEV),
                            torch.stack([a[1] for a in _adapters(3, n, k, [5] * 3, 2)]).to(DEV),
                            torch.tensor([a[2] for a in _adapters(3, n, k, [5] * 3, 2)], device=DEV))
    _check(kernels.lora_add(dy, dx, again, di), y, x, _adapters(3, n, k, [5] * 3, 2), index)


@pytest.mark.parametrize("m", [1, 9, 70])
def test_lora_linear(gpu, m):
    """The whole projection in its three forms: the shared part as linear()
    rounds it, then the adapters; rows without one are bit for bit linear()'s."""
    n, k = 512, 1024
    x, res = seeded_normal((m, k), 1.0, 1), seeded_normal((m, n), 1.0, 2)
    w = seeded_normal((n, k), 0.02, 3)
    adapters = _adapters(3, n, k, [8, 16, 12], seed=4)
    index = _index(m, 3, 6)
    dx, di, plain = x.to(DEV), index.to(DEV), index < 0
    weight = PackedWeight.from_rowmajor(w.to(DEV))
    store = _store(adapters, n, k, 16)
    for kw in ({}, {"epilogue": _lib.EPI_RESIDUAL_ADD, "residual": res.to(DEV)}):
        base = kernels.linear(dx, weight, **kw)
        got = kernels.lora_linear(dx, weight, store, di, **kw)
        _check(got, base.cpu(), x, adapters, index)
        assert torch.equal(got.cpu()[plain], base.cpu()[plain])
        out = torch.empty_like(base)
        assert kernels.lora_linear(dx, weight, store, di, out=out, **kw) is out and torch.equal(out, got)
    gu = PackedWeight.from_rowmajor(w.to(DEV), _lib.LAYOUT_MFMA16X32_GATEUP)
    rows = torch.arange(n).view(2, n // 32, 16).transpose(0, 1).reshape(-1)
    both = kernels.linear(dx, PackedWeight(gu.data, n, k))
    assert torch.equal(both[:, :16], kernels.linear(dx, weight)[:, :16])
    got = kernels.lora_linear(dx, gu, _store(adapters, n, k, 16, gate_up=True), di, epilogue=SILU)
    _check(got, both.cpu(), x, [(a, b[rows], s) for a, b, s in adapters], index, gate_up=True)


def test_parts_of_a_fused_projection(gpu):
    """Adapters of q, k and v side by side are those of the three projections."""
    k, sizes, m = 256, (128, 32, 32), 6
    n = sum(sizes)
    parts = [_adapters(1, s, k, [r], seed=s + r)[0][:2] for s, r in zip(sizes, (8, 8, 5))]
    store = AdapterStore(1, n, k, 21, device=DEV)
    store.load_parts(0, [(a.to(DEV), b.to(DEV)) for a, b in parts], 2.0)
    y, x = seeded_normal((m, n), 1.0, 1), seeded_normal((m, k), 1.0, 2)
    index = torch.zeros(m, dtype=torch.int32)
    got = kernels.lora_add(y.to(DEV), x.to(DEV), store, index.to(DEV)).cpu()
    at = 0
    for (a, b), s in zip(parts, sizes):
        _check(got[:, at:at + s], y[:, at:at + s], x, [(a, b, 2.0)], index)
        at += s


@pytest.mark.parametrize("m,k,rank", [(20, 512, 16), (20, 9728, 64), (200, 512, 16)])
def test_captured_and_on_two_streams(gpu, m, k, rank):
    """Replays follow the index, the rows and the store's slots as they are then;
    calls on two streams at once share nothing."""
    n, count = 640, 4
    adapters = _adapters(count, n, k, [rank] * count, seed=3)
    store, other = _store(adapters, n, k, rank), _store(adapters[::-1], n, k, rank)
    ys = [seeded_normal((m, n), 1.0, s).to(DEV) for s in (1, 2)]
    xs = [seeded_normal((m, k), 1.0, s).to(DEV) for s in (3, 4)]
    ids = [_index(m, count, s).to(DEV) for s in (5, 6)]
    y, x, index = ys[0].clone(), xs[0].clone(), ids[0].clone()
    kernels.lora_add(y, x, store, index)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, kernels.lora_add(y, x, store, index)))
    for step in range(4):
        y.copy_(ys[step % 2]), x.copy_(xs[step // 2]), index.copy_(ids[step % 2])
        if step == 2:
            store.load(1, adapters[0][0].to(DEV), adapters[2][1].to(DEV), 0.75)
        expect = kernels.lora_add(y, x, store, index)
        for graph, out in graphs:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, expect)
    pairs = [(ys[0], xs[0], store, ids[0]), (ys[1], xs[1], other, ids[1])]
    expect = [kernels.lora_add(*p) for p in pairs]
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(5):
        for stream, p in zip(streams, pairs):
            with torch.cuda.stream(stream):
                results.append(kernels.lora_add(*p))
    torch.cuda.synchronize()
    for i, out in enumerate(results):
        assert torch.equal(out, expect[i % 2])
