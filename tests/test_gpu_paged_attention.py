"""Attention over the pages of an 8-bit cache on the GPU, value by value against its definition in 64 bits."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from leanstack_amd import kernels
from leanstack_amd.paged_cache import PagedKVCache

from paged_helpers import D, Pool, attention, number

pytestmark = pytest.mark.gpu


def ints(gpu, values):
    return torch.tensor(values, dtype=torch.int32, device=gpu)


def setup(gpu, n_kv, page_rows, lens, seed, spare=2, std=1.0):
    """A layer of normal values with an exponent that differs from block to block, NaN and wild exponents in every
    page and block that no request's rows reach, and the table of the requests."""
    rng = np.random.default_rng(seed)
    need = [max(0, -(-n // page_rows)) for n in lens]
    pages = sum(need) + spare
    blocks = page_rows // 16
    shape = (1, 2, pages, n_kv, blocks)
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((*shape, 16 * D), generator=gen) * std
    e = torch.randint(-9, -5, shape, generator=gen)
    storage = (x * torch.exp2(-e.float())[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    exponents = (e + 127).to(torch.uint8)
    order = rng.permutation(pages)
    width = max([1] + need) + 1
    table = [[-1] * width for _ in lens]
    used = 0
    for b, n in enumerate(need):
        table[b][:n] = order[used:used + n].tolist()
        used += n
    # what stands behind the rows is not read
    from paged_helpers import places
    stale = torch.zeros((2, pages, blocks, 16), dtype=torch.bool)
    stale[:] = True
    for b, n in enumerate(lens):
        for r in range(max(n, 0)):
            stale[:, table[b][r // page_rows], r % page_rows // 16, r % 16] = False
    for kv in range(2):
        at = torch.from_numpy(places()[kv])
        for page, block in stale[kv].any(-1).nonzero().tolist():
            rows = stale[kv, page, block]
            storage[0, kv, page, :, block][:, at[rows].reshape(-1)] = 0x7F
            if bool(rows.all()):
                exponents[0, kv, page, :, block] = 255
    cache = PagedKVCache.of(storage.to(gpu), exponents.to(gpu))
    return cache, table


def queries(b, n_q, t, seed, std=1.5):
    return (torch.randn((b, n_q, t, D), generator=torch.Generator().manual_seed(seed)) * std).to(torch.bfloat16)


def check(gpu, cache, q, table, lens, scale, counts=None, **kwargs):
    got = kernels.paged_attention(q.to(gpu), cache, 0, ints(gpu, table), ints(gpu, lens), scale,
                                  counts=None if counts is None else ints(gpu, counts), **kwargs)
    b, n_q, t, _ = q.shape
    assert got.shape == (b, t, n_q * D) and got.dtype is torch.bfloat16
    want, bound = attention(Pool(cache.storage[0], cache.exponents[0]), q, table, lens, scale, counts)
    got = got.cpu().double().view(b, t, n_q, D)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    off = torch.where(nan, 0, (got - want).abs())
    over = off > torch.where(nan, 1, bound)
    assert not bool(over.any()), f"{int(over.sum())} values off, worst {float((off / bound).max())} of the bound"
    return got


@pytest.mark.parametrize("n_q,n_kv,page_rows,t,lens,counts", [
    (32, 8, 64, 1, [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65], None),      # single tokens, all ends of blocks and steps
    (32, 8, 64, 1, [0, -3, 1000, 129, 700], None),                         # none; several steps per wave
    (8, 1, 16, 1, [5, 500, 48], None),
    (1, 1, 16, 1, [37], None),
    (16, 16, 32, 1, [100, 1, 257], None),                                  # a q head per kv head
    (6, 2, 128, 1, [300, 128], None),                                      # groups of 3
    (40, 8, 64, 1, [200, 77], None),                                       # groups of 5
    (48, 2, 64, 1, [90], None),                                            # groups of 24: two tiles of query rows
    (32, 8, 32, 5, [5, 6, 33, 500, 36], None),                             # verify blocks
    (32, 8, 64, 5, [5, 40, 64, 0, 200], [5, 0, 3, 2, 1]),                  # padded, one without rows, one empty
    (32, 8, 64, 4, [2, 3, 4, 1], None),                                    # fewer rows than queries: the first see none
    (8, 4, 16, 16, [16, 47, 30], [16, 16, 9]),
    (8, 1, 64, 8, [100, 8], None),                                         # 64 query rows of a kv head
    (12, 4, 16, 7, [19, 7, 300], None),                                    # 21 query rows
    (32, 8, 64, 33, [33, 100, 64], [33, 20, 33]),                          # prompts: several tiles
    (4, 2, 32, 300, [300, 421], [300, 111]),
    (8, 1, 128, 130, [1500, 130], None),
    (2, 1, 1024, 3, [2100, 1024, 1025], None),
])
def test_sizes(gpu, n_q, n_kv, page_rows, t, lens, counts):
    cache, table = setup(gpu, n_kv, page_rows, lens, seed=len(lens) + t)
    q = queries(len(lens), n_q, t, seed=t + n_q)
    got = check(gpu, cache, q, table, lens, D ** -0.5, counts)
    for b, n in enumerate(lens):
        count = t if counts is None else counts[b]
        for j in range(t):
            if j >= count or max(n, 0) - (count - 1 - j) <= 0:
                assert not got[b, j].any()


@pytest.mark.parametrize("t,n_q,n_kv", [(1, 32, 8), (1, 8, 1), (3, 8, 2), (40, 4, 1)])
def test_long(gpu, t, n_q, n_kv):
    """Contexts over which the rows are split, ragged."""
    lens = [9000, 40, 3333, 6001]
    cache, table = setup(gpu, n_kv, 64, lens, seed=31)
    check(gpu, cache, queries(4, n_q, t, seed=32), table, lens, D ** -0.5)


def test_many_requests(gpu):
    lens = [(37 * i) % 150 for i in range(130)]
    cache, table = setup(gpu, 2, 16, lens, seed=33)
    check(gpu, cache, queries(130, 8, 1, seed=34), table, lens, D ** -0.5)
    check(gpu, cache, queries(130, 8, 2, seed=35), table, lens, D ** -0.5, [i % 3 for i in range(130)])


@pytest.mark.parametrize("t,n_q", [(1, 4), (5, 4), (90, 2)])
def test_a_million_rows(gpu, t, n_q):
    """A context of 2^20 rows, of 16 pages named again and again: the result is that of rows which
    all weigh as often as they are named (the last, begun round aside, whose rows are left out).
    Sums of 2^20 weights in fp32, in chunks: 2^-24 for each of a chunk's, at most 2^14 in a row."""
    n_kv, page_rows, pages = 1, 64, 16
    cache, table = setup(gpu, n_kv, page_rows, [pages * page_rows], seed=31)
    named = table[0][:pages]
    rounds = 1024
    q = queries(1, n_q, t, seed=32)
    # the same rows for every query token: the last rounds have no page
    wide = named * rounds + [-1] * (t // page_rows + 1)
    got = kernels.paged_attention(q.to(gpu), cache, 0, ints(gpu, [wide]), ints(gpu, [pages * page_rows * rounds + t - 1]), 0.1)
    pool = Pool(cache.storage[0], cache.exponents[0])
    for i in range(t):
        want, bound = attention(pool, q[:, :, i:i + 1], [named], [pages * page_rows], 0.1)
        most = pool.dense(named, pages * page_rows)[1].abs().max()
        off = (got[:, i].cpu().double().view(1, 1, n_q, D) - want).abs()
        assert bool((off <= bound + 2 * 2.0 ** -10 * most).all())


@pytest.mark.parametrize("n_q,n_kv,t,lens,counts", [
    (4, 1, 1, [16500], None), (32, 8, 1, [9000, 33, 0, 2500], None), (3, 1, 1, [20000, 7], None),   # many parts of few rows
    (4, 1, 5, [17000], None), (8, 2, 5, [5000, 3, 2100, 5], [5, 3, 4, 0]), (2, 2, 32, [2100, 40], None),
    (4, 1, 10, [3000], None), (8, 2, 16, [2300, 16, 9], [16, 16, 3]),   # 33..64 rows in two launches
    (4, 1, 20, [9000], None), (2, 1, 33, [8500, 12], [33, 1]),          # .. many parts of them
    (32, 8, 128, [128, 300, 129, 5, 192, 200, 128, 130, 131], [128, 128, 128, 5, 128, 100, 1, 128, 0]),
    (64, 8, 17, [17 + 11 * i % 150 for i in range(70)], None),          # more items than workers, short and cut ones
    (32, 8, 150, [150, 700, 151, 0, 160, 170, 155, 900, 150, 180, 200, 151], [150, 150, 9, 0, 150, 1, 150, 150, 40, 150, 150, 150]),
    (4, 4, 1, [33 + 8 * i for i in range(140)], None), (8, 8, 3, [33 + 8 * i for i in range(70)], None),  # whole and cut ones
])
def test_parts(gpu, n_q, n_kv, t, lens, counts):
    """Contexts cut into any number of parts, joined by workgroups of each kind."""
    cache, table = setup(gpu, n_kv, 64, lens, seed=41)
    wide = [row + [-1] * 33 for row in table]   # (a table of more than 2048 rows: no call in one launch)
    check(gpu, cache, queries(len(lens), n_q, t, seed=42), wide, lens, 0.1, counts)


@pytest.mark.parametrize("t", [1, 6, 70])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 1.0, 1e-30, 40.0])
def test_scales(gpu, t, scale):
    """Any sign; weights all alike; and scores so far apart that one row has all the weight."""
    lens = [100, 333]
    cache, table = setup(gpu, 2, 32, lens, seed=36)
    check(gpu, cache, queries(2, 8, t, seed=37), table, lens, scale)


@pytest.mark.parametrize("t", [1, 6, 70])
@pytest.mark.parametrize("size", [1e20, 1e30])
def test_far_scores(gpu, t, size):
    """Scores beyond what a difference of rounded exponents can hold: the largest takes all."""
    lens = [100, 333]
    cache, table = setup(gpu, 2, 32, lens, seed=38)
    q = (queries(2, 8, t, seed=39).float() * size).to(torch.bfloat16)
    pool = Pool(cache.storage[0], cache.exponents[0])
    got = kernels.paged_attention(q.to(gpu), cache, 0, ints(gpu, table), ints(gpu, lens), 1.0).cpu().double().view(2, t, 8, D)
    want, _ = attention(pool, q, table, lens, 1.0)
    assert float((got - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())


@pytest.mark.parametrize("t,at", [(1, 5), (1, 199), (3, 198), (3, 50), (80, 130), (80, 10), (80, 199)])
def test_nan_rows(gpu, t, at):
    """A value row with a NaN reaches the queries that see it and no other; a key row likewise, in every value."""
    lens = [200, 200]
    for what in ("v", "k"):
        cache, table = setup(gpu, 2, 32, lens, seed=40)
        page, row = table[0][at // 32], at % 32
        from paged_helpers import places
        kv = 1 if what == "v" else 0
        cache.storage[0, kv, page, 1, row // 16, int(places()[kv][row % 16, 77])] = 0x7F
        q = queries(2, 8, t, seed=41)
        got = kernels.paged_attention(q.to(gpu), cache, 0, ints(gpu, table), ints(gpu, lens), D ** -0.5).cpu().view(2, t, 8, D)
        seen = torch.tensor([200 - (t - 1 - j) > at for j in range(t)])
        nan = torch.zeros_like(got, dtype=torch.bool)
        nan[0, :, 4:, 77 if what == "v" else slice(None)] = seen[:, None] if what == "v" else seen[:, None, None]
        assert torch.equal(torch.isnan(got), nan)
        pool = Pool(cache.storage[0], cache.exponents[0])
        pool.bytes[kv, page, 1, row // 16, places()[kv][row % 16, 77]] = 0
        want, bound = attention(pool, q, table, lens, D ** -0.5)
        fine = ~nan if what == "v" else ~seen[None, :, None, None].expand_as(nan)
        assert bool(((got.double() - want).abs() <= bound)[fine].all())


def test_infinite_query(gpu):
    """Scores that are all -inf, or NaN, give NaN, and only for their own query."""
    lens = [60]
    cache, table = setup(gpu, 1, 64, lens, seed=42)
    cache.storage[0, 0, :, :, :, :] = 0x38  # keys of ones
    cache.exponents[0, 0] = 127
    q = torch.ones((1, 4, 1, D), dtype=torch.bfloat16)
    q[0, 1, 0, 3], q[0, 2, 0, 3], q[0, 3, 0, 5] = -float("inf"), float("inf"), float("nan")
    got = kernels.paged_attention(q.to(gpu), cache, 0, ints(gpu, table), ints(gpu, lens), 1.0).cpu().view(4, D)
    assert torch.isnan(got[1:]).all() and torch.isfinite(got[0]).all()


def test_entries_that_name_no_page(gpu):
    """Rows there are seen by no query; a query that sees no other gives zeros."""
    lens = [150, 64, 40]
    cache, table = setup(gpu, 2, 16, lens, seed=43, spare=0)
    table[0][0], table[0][4], table[0][9] = -1, cache.num_pages, -(1 << 31)
    table[2] = [1 << 30] * len(table[2])
    for t in (1, 5, 40):
        got = check(gpu, cache, queries(3, 8, t, seed=44), table, lens, D ** -0.5)
        assert not got[2].any()


def test_lens_past_the_table(gpu):
    lens = [64, 30]
    cache, table = setup(gpu, 2, 16, lens, seed=45)
    table = [row[:4] for row in table]
    for t in (1, 5, 90):
        check(gpu, cache, queries(2, 4, t, seed=46), table, [70, 1 << 30], D ** -0.5, None)


def test_shared_pages(gpu):
    """Two requests over the same pages."""
    lens = [100, 0]
    cache, table = setup(gpu, 2, 16, lens, seed=47)
    table[1] = list(table[0])
    check(gpu, cache, queries(2, 8, 2, seed=48), table, [100, 61], D ** -0.5)


def test_strides_and_out(gpu):
    """Queries as views and copies give the same bits; `out` is written whole and nothing beside it."""
    lens = [70, 33]
    cache, table = setup(gpu, 4, 32, lens, seed=49)
    q = queries(2, 8, 3, seed=50).to(gpu)
    args = (cache, 0, ints(gpu, table), ints(gpu, lens), D ** -0.5)
    want = kernels.paged_attention(q, *args)
    rows = torch.zeros((2, 3, 24, D), dtype=torch.bfloat16, device=gpu)
    rows[:, :, 4:12] = q.transpose(1, 2)
    odd = torch.zeros(q.numel() + 1, dtype=torch.bfloat16, device=gpu)[1:].view_as(q)
    odd.copy_(q)
    for same in (rows[:, :, 4:12].transpose(1, 2), odd, q.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(kernels.paged_attention(same, *args), want)
    wide = torch.full((4, 3, 8 * D), 7.0, dtype=torch.bfloat16, device=gpu)
    got = kernels.paged_attention(q, *args, out=wide[1:3])
    assert got.data_ptr() == wide[1:3].data_ptr() and torch.equal(got, want) and bool((wide[0] == 7).all() and (wide[3] == 7).all())
    table_view = torch.full((2, len(table[0]) + 5), 99, dtype=torch.int32, device=gpu)[:, :len(table[0])]
    table_view.copy_(ints(gpu, table))
    assert torch.equal(kernels.paged_attention(q, cache, 0, table_view, ints(gpu, lens), D ** -0.5), want)


def test_same_bits_every_time(gpu):
    lens = [5000, 17, 2222]
    cache, table = setup(gpu, 8, 64, lens, seed=51)
    for t in (1, 5):
        q = queries(3, 32, t, seed=52).to(gpu)
        args = (q, cache, 0, ints(gpu, table), ints(gpu, lens), D ** -0.5)
        want = kernels.paged_attention(*args)
        for _ in range(20):
            assert torch.equal(kernels.paged_attention(*args), want)


@pytest.mark.parametrize("t", [1, 5, 48])
def test_captured(gpu, t):
    """Replays follow lens, counts and the table, beside eager calls on the same stream."""
    lens = [900, 333]
    cache, table = setup(gpu, 2, 64, lens, seed=53)
    q = queries(2, 8, t, seed=54).to(gpu)
    where, now, counts = ints(gpu, table), ints(gpu, lens), ints(gpu, [t, t])
    kernels.paged_attention(q, cache, 0, where, now, D ** -0.5, counts=counts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kernels.paged_attention(q, cache, 0, where, now, D ** -0.5, counts=counts)
        again = kernels.paged_attention(q, cache, 0, where, now, 0.05)
    for rows, new in (([900, 333], [t, t]), ([10, 0], [t, 1]), ([500, 64], [max(1, t - 1), t]), ([899, 100], [1, 0])):
        now.copy_(ints(gpu, rows)), counts.copy_(ints(gpu, new))
        graph.replay()
        eager = kernels.paged_attention(q, cache, 0, where, now, D ** -0.5, counts=counts)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        assert torch.equal(again, kernels.paged_attention(q, cache, 0, where, now, 0.05, counts=None))


def test_streams(gpu):
    """Calls that overlap on two streams."""
    lens = [3000, 500, 2000]
    cache, table = setup(gpu, 8, 64, lens, seed=55)
    where, now = ints(gpu, table), ints(gpu, lens)
    fed = [queries(3, 32, 1, seed=56 + i).to(gpu) for i in range(4)]
    want = [kernels.paged_attention(q, cache, 0, where, now, D ** -0.5) for q in fed]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[] for _ in fed]
    for _ in range(10):
        for i, q in enumerate(fed):
            with torch.cuda.stream(streams[i % 2]):
                got[i].append(kernels.paged_attention(q, cache, 0, where, now, D ** -0.5))
    torch.cuda.synchronize()
    for i in range(4):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_stale_numbers_are_what_the_helper_says():
    assert np.isnan(number(np.array([0x7F, 0xFF], dtype=np.uint8))).all() and math.isclose(float(number(np.array([0x38]))[0]), 1.0)
