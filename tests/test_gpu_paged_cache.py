"""The paged 8-bit cache on the GPU: rows in, rows out and pages copied, byte by byte against the format's definition."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from leanstack_amd import kernels
from leanstack_amd.kv_cache import ArenaKVCache
from leanstack_amd.paged_cache import PagedKVCache

from paged_helpers import E4M3, Pool

pytestmark = pytest.mark.gpu


def random_pool(gpu, layers, n_kv, pages, page_rows, seed):
    """A pool of any bytes, NaN and odd exponents among them."""
    gen = torch.Generator().manual_seed(seed)
    shape = (layers, 2, pages, n_kv, page_rows // 16)
    storage = torch.randint(0, 256, (*shape, 2048), generator=gen, dtype=torch.uint8)
    exponents = torch.randint(100, 150, shape, generator=gen, dtype=torch.uint8)
    return PagedKVCache.of(storage.to(gpu), exponents.to(gpu))


def new_rows(b, n_kv, t, seed):
    """Rows whose sizes differ from row to row by powers of two, zeros among them."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((2, b, n_kv, t, 128), generator=gen)
    x *= torch.exp2(torch.randint(-12, 6, (2, b, n_kv, t, 1), generator=gen).float())
    x *= (torch.rand((2, b, n_kv, t, 1), generator=gen) > 0.1).float()
    x = x.to(torch.bfloat16)
    return x[0], x[1]


def same(cache, pool, layer=0):
    """The layer's bytes (as numbers: NaN equal to NaN, -0 to 0) and exponents are the pool's."""
    got = Pool(cache.storage[layer], cache.exponents[layer])
    from paged_helpers import number
    np.testing.assert_array_equal(got.exponents, pool.exponents)
    np.testing.assert_array_equal(number(got.bytes), number(pool.bytes))


def tables(gpu, rows):
    return torch.tensor(rows, dtype=torch.int32, device=gpu)


def ints(gpu, values):
    return torch.tensor(values, dtype=torch.int32, device=gpu)


@pytest.mark.parametrize("page_rows,n_kv,t,lens,counts", [
    (64, 8, 1, [1, 16, 17, 64, 65, 150], None),           # single rows: the first, the last of a block, of a page, behind one
    (16, 1, 1, [5, 33], None),
    (32, 2, 5, [5, 16, 20, 35, 64], None),                # verify blocks that end, start and cross blocks
    (64, 3, 15, [15, 30, 79], [15, 0, 7]),                # padded, one with nothing new
    (16, 2, 16, [16, 40], None),
    (64, 1, 17, [17, 33, 100], None),
    (128, 2, 100, [100, 131, 250], [100, 99, 1]),
    (1024, 1, 33, [1056, 33], None),                      # the largest page
    (32, 2, 8, [3, 0, -4, 8], None),                      # rows in front of row 0 are dropped
    (16, 2, 40, [40, 70, 100], [39, 40, 1000]),           # rows past the table are dropped; a count beyond T is T
])
def test_append_is_the_definition(gpu, page_rows, n_kv, t, lens, counts):
    pages = 4 * len(lens) + 1
    cache = random_pool(gpu, 2, n_kv, pages, page_rows, seed=t)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
    table = [order[4 * i:4 * i + 4] for i in range(len(lens))]
    pool, other = Pool(cache.storage[1], cache.exponents[1]), Pool(cache.storage[0], cache.exponents[0])
    k, v = new_rows(len(lens), n_kv, t, seed=7 * t + page_rows)
    for again in range(2):  # the same call twice leaves the same
        kernels.paged_append(cache, 1, k.to(gpu), v.to(gpu), tables(gpu, table), ints(gpu, lens),
                             counts=None if counts is None else ints(gpu, counts))
        if not again:
            pool.append(k, v, table, lens, counts)
        same(cache, pool, 1)
    same(cache, other, 0)


def test_row_after_row(gpu):
    """A block filled row by row, its exponent rising and its rows rounded again, or not."""
    cache = random_pool(gpu, 1, 2, 3, 32, seed=3)
    pool = Pool(cache.storage[0], cache.exponents[0])
    table = [[2, 0]]
    for i in range(40):
        k, v = new_rows(1, 2, 1, seed=100 + i)
        kernels.paged_append(cache, 0, k.to(gpu), v.to(gpu), tables(gpu, table), ints(gpu, [i + 1]))
        pool.append(k, v, table, [i + 1])
    same(cache, pool)


def test_every_bf16_value(gpu):
    """All 2^16 bit patterns, in blocks of like size (one exponent each), and alone at the head of a block."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    k = bits.view(1, 1, 512, 128)
    order = torch.randperm(1 << 16, generator=torch.Generator().manual_seed(5))
    v = bits[order].view(1, 1, 512, 128)
    cache = random_pool(gpu, 1, 1, 8, 64, seed=4)
    pool = Pool(cache.storage[0], cache.exponents[0])
    table = [[3, 1, 0, 2, 7, 5, 6, 4]]
    kernels.paged_append(cache, 0, k.to(gpu), v.to(gpu), tables(gpu, table), ints(gpu, [512]))
    pool.append(k, v, table, [512])
    same(cache, pool)


@pytest.mark.parametrize("e", [-100, -99, -20, 0, 50, 118, 119])
def test_ties_and_ends_of_the_exponents(gpu, e):
    """Values half way between two stored ones (ties to even), the largest of an exponent, one step above it."""
    steps = E4M3[:-1] + np.diff(E4M3) / 2
    values = np.concatenate([steps, -steps, [448, 449, 0, -0.0, 2.0 ** -10, 2.0 ** -11]])
    with np.errstate(over="ignore"):
        x = torch.from_numpy(np.resize(values, (1, 1, 34, 128)) * 2.0 ** e).to(torch.bfloat16)
    x[0, 0, 16:32] = torch.where(x[0, 0, 16:32].abs() > 448 * 2.0 ** e, 0, x[0, 0, 16:32])
    cache = random_pool(gpu, 1, 1, 1, 64, seed=6)
    pool = Pool(cache.storage[0], cache.exponents[0])
    kernels.paged_append(cache, 0, x.to(gpu), (-x).to(gpu), tables(gpu, [[0]]), ints(gpu, [34]))
    pool.append(x, -x, [[0]], [34])
    same(cache, pool)


def test_infinities_and_nan(gpu):
    """They become NaN, and say nothing about the block's exponent; a block of nothing else, and one of zeros."""
    k, v = new_rows(1, 1, 64, seed=8)
    k[0, 0, 3, 5], k[0, 0, 4, 127], v[0, 0, 0, 0], v[0, 0, 15, 16] = float("inf"), float("nan"), -float("inf"), float("nan")
    k[0, 0, 16:32], v[0, 0, 16:32], k[0, 0, 32:48], v[0, 0, 32:48] = float("nan"), float("inf"), 0, -0.0
    cache = random_pool(gpu, 1, 1, 1, 64, seed=9)
    pool = Pool(cache.storage[0], cache.exponents[0])
    table = tables(gpu, [[0]])
    for n in (20, 64):  # the second call goes on in a block that holds NaN
        first = 0 if n == 20 else 20
        kernels.paged_append(cache, 0, k[:, :, first:n].to(gpu), v[:, :, first:n].to(gpu), table, ints(gpu, [n]))
        pool.append(k[:, :, first:n], v[:, :, first:n], [[0]], [n])
    same(cache, pool)


def test_entries_that_name_no_page(gpu):
    """Rows there are dropped, and read back as zeros; the others are kept."""
    cache = random_pool(gpu, 1, 2, 3, 16, seed=10)
    pool = Pool(cache.storage[0], cache.exponents[0])
    table = [[0, -1, 2, 3, 1 << 30], [-(1 << 31), 1, 5, -7, -1]]
    k, v = new_rows(2, 2, 70, seed=11)
    kernels.paged_append(cache, 0, k.to(gpu), v.to(gpu), tables(gpu, table), ints(gpu, [70, 75]))
    pool.append(k, v, table, [70, 75])
    same(cache, pool)
    got = kernels.paged_read(cache, 0, tables(gpu, table), ints(gpu, [0, 0]), 80, lens=ints(gpu, [70, 75]))
    for kv in range(2):
        for b, n in enumerate((70, 75)):
            for head in range(2):
                want = pool.rows(kv, table[b], head, 0, 80)
                want[n:] = 0
                np.testing.assert_array_equal(got[kv][b, head].double().cpu().numpy(), want)


@pytest.mark.parametrize("starts,rows,lens", [([0, 5, 40], 33, [33, 38, 64]), ([63, 0, 1], 1, [64, 0, 1]),
                                              ([16, -3, 200], 64, None), ([7, 8, 9], 17, [1 << 30, -5, 20])])
def test_read(gpu, starts, rows, lens):
    cache = random_pool(gpu, 2, 3, 7, 32, seed=12)
    table = [[0, 3], [6, 1], [5, 5]]
    pool = Pool(cache.storage[1], cache.exponents[1])
    got = kernels.paged_read(cache, 1, tables(gpu, table), ints(gpu, starts), rows, lens=None if lens is None else ints(gpu, lens))
    for kv in range(2):
        assert got[kv].shape == (3, 3, rows, 128) and got[kv].dtype is torch.bfloat16
        for b in range(3):
            first = max(starts[b], 0)
            for head in range(3):
                want = pool.rows(kv, table[b], head, first, rows)
                if lens is not None:
                    want[max(max(lens[b], 0) - first, 0):] = 0
                np.testing.assert_array_equal(got[kv][b, head].double().cpu().numpy(), want)


def test_any_strides(gpu):
    """Views of projection rows, a misaligned start and strides that need a copy give what contiguous rows give."""
    b, n_kv, t = 2, 4, 21
    qkv = torch.randn((b, t, 12, 128), device=gpu).to(torch.bfloat16)
    k, v = qkv[:, :, 4:8].transpose(1, 2), qkv[:, :, 8:].transpose(1, 2)
    odd = torch.randn(b * n_kv * t * 129 + 1, device=gpu).to(torch.bfloat16)[1:].view(b, n_kv, t, 129)[..., :128]
    table, lens = tables(gpu, [[0, 1, 2], [5, 4, 3]]), ints(gpu, [40, 21])
    for keys, values in ((k, v), (odd, v), (k.transpose(2, 3).contiguous().transpose(2, 3), odd)):
        one, two = random_pool(gpu, 1, n_kv, 6, 16, seed=13), random_pool(gpu, 1, n_kv, 6, 16, seed=13)
        kernels.paged_append(one, 0, keys, values, table, lens)
        kernels.paged_append(two, 0, keys.contiguous().clone(), values.contiguous().clone(), table, lens)
        assert torch.equal(one.storage, two.storage) and torch.equal(one.exponents, two.exponents)


def test_copy_pages(gpu):
    """All layers; entries outside the pool copy nothing; other pages stay."""
    cache = random_pool(gpu, 3, 2, 9, 64, seed=14)
    storage, exponents = cache.storage.clone(), cache.exponents.clone()
    kernels.copy_pages(cache, ints(gpu, [0, 8, 3, -1, 4, 9]), ints(gpu, [5, 1, 2, 6, -1, 7]))
    for src, dst in ((0, 5), (8, 1), (3, 2)):
        storage[:, :, dst], exponents[:, :, dst] = storage[:, :, src].clone(), exponents[:, :, src].clone()
    assert torch.equal(cache.storage, storage) and torch.equal(cache.exponents, exponents)
    kernels.copy_pages(cache, ints(gpu, []), ints(gpu, []))
    assert torch.equal(cache.storage, storage)


@pytest.mark.parametrize("n_kv,page_rows", [(1, 16), (5, 16), (3, 1024), (8, 64)])
def test_copy_whole_pages_of_any_size(gpu, n_kv, page_rows):
    cache = random_pool(gpu, 1, n_kv, 4, page_rows, seed=15)
    storage, exponents = cache.storage.clone(), cache.exponents.clone()
    kernels.copy_pages(cache, ints(gpu, [1]), ints(gpu, [3]))
    storage[:, :, 3], exponents[:, :, 3] = storage[:, :, 1].clone(), exponents[:, :, 1].clone()
    assert torch.equal(cache.storage, storage) and torch.equal(cache.exponents, exponents)


def test_pages_past_four_gib(gpu):
    """Rows, copies and attention in pages whose bytes lie past 2^32 of a layer's keys, as in a small pool."""
    n_kv, page_rows, far, middle = 8, 1024, 4299, 2100
    large, small = PagedKVCache(1, n_kv, far + 1, page_rows=page_rows, device=gpu), PagedKVCache(1, n_kv, 4, page_rows=page_rows, device=gpu)
    where, lens = {0: far, 1: middle, 2: far - 1, 3: 7}, [1000, 1500]
    k, v = (x.to(gpu) for x in new_rows(2, n_kv, 700, seed=40))
    q = new_rows(2, 4 * n_kv, 40, seed=41)[0].to(gpu)
    results = []
    for cache, name in ((small, lambda p: p), (large, lambda p: where[p])):
        table = tables(gpu, [[name(0), name(1)], [name(2), name(3)]])
        kernels.paged_append(cache, 0, k, v, table, ints(gpu, lens))
        kernels.copy_pages(cache, ints(gpu, [name(0)]), ints(gpu, [name(1)]))
        results.append([*kernels.paged_read(cache, 0, table, ints(gpu, [300, 800]), 1200), *(
            kernels.paged_attention(q[:, :, :t].contiguous(), cache, 0, table, ints(gpu, lens), 0.1) for t in (1, 7, 40))])
    assert all(torch.equal(x, y) for x, y in zip(*results))
    for p, at in where.items():
        assert torch.equal(small.storage[:, :, p], large.storage[:, :, at])
        assert torch.equal(small.exponents[:, :, p], large.exponents[:, :, at])
    others = [p for p in (0, 1, 2, 3, 4, 5, 6, 8, middle - 1, middle + 1, far - 2)]
    assert not bool(large.storage[:, :, others].any())


def test_captured_append_follows_lens_counts_and_table(gpu):
    cache = random_pool(gpu, 1, 2, 6, 16, seed=16)
    pool = Pool(cache.storage[0], cache.exponents[0])
    table, lens, counts = tables(gpu, [[0, 1], [2, 3]]), ints(gpu, [3, 3]), ints(gpu, [3, 2])
    k, v = (x.to(gpu) for x in new_rows(2, 2, 3, seed=17))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.paged_append(cache, 0, k, v, table, lens, counts=counts)
        back = kernels.paged_read(cache, 0, table, lens - counts, 3, lens=lens)
    same(cache, pool)  # (a capture runs nothing)
    for step, (rows, now, new) in enumerate((([[0, 1], [2, 3]], [3, 3], [3, 2]), ([[0, 1], [4, 3]], [6, 18], [3, 3]),
                                             ([[5, 1], [4, 3]], [1, 20], [0, 2]))):
        fresh = new_rows(2, 2, 3, seed=18 + step)
        k.copy_(fresh[0]), v.copy_(fresh[1]), table.copy_(tables(gpu, rows)), lens.copy_(ints(gpu, now)), counts.copy_(ints(gpu, new))
        graph.replay()
        pool.append(*fresh, rows, now, new)
        same(cache, pool)
        want = pool.rows(0, rows[1], 0, now[1] - new[1], new[1])
        np.testing.assert_array_equal(back[0][1, 0, :new[1]].double().cpu().numpy(), want)


def test_requests_fork_grow_and_compact(gpu):
    """What each request reads back stays its own through shared pages, copies, cuts and moves."""
    layers, n_kv = 2, 2
    cache = PagedKVCache(layers, n_kv, 12, page_rows=16, device=gpu)
    kept: dict[int, list] = {}

    def grow(requests, n, seed):
        cache.reserve(requests, n)
        table, lens = cache.batch(requests, n)
        for layer in range(layers):
            k, v = new_rows(len(requests), n_kv, n, seed=seed + layer)
            kernels.paged_append(cache, layer, k.to(gpu), v.to(gpu), table, lens)
        cache.advance(requests, n)

    def read(r):
        table, lens = cache.batch([r])
        return [torch.stack(kernels.paged_read(cache, layer, table, torch.zeros_like(lens), r.rows, lens=lens))
                for layer in range(layers)]

    a = cache.open()
    grow([a], 21, seed=50)
    first = read(a)
    b, c = cache.fork(a), cache.fork(a)
    assert cache.free_pages == 10
    grow([a, b, c], 3, seed=60)  # two copies of the begun page: the last to write keeps it
    assert cache.free_pages == 8 and len({r.pages[1] for r in (a, b, c)}) == 3
    for r in (a, b, c):
        kept[id(r)] = read(r)
        # rows of shared blocks may have been rounded again; whole blocks in front of them are as they were
        assert all(torch.equal(x[..., :16, :], y[..., :16, :]) for x, y in zip(kept[id(r)], first))
    cache.truncate(b, 18)
    cache.close(a)
    grow([c], 30, seed=70)
    kept[id(c)] = read(c)
    used = cache.compact()
    assert used == len({p for r in (b, c) for p in r.pages}) and max(p for r in (b, c) for p in r.pages) < used
    assert all(torch.equal(x[..., :18, :], y) for x, y in zip(kept[id(b)], read(b)))
    assert all(torch.equal(x, y) for x, y in zip(kept[id(c)], read(c)))
    arena = ArenaKVCache(layers, n_kv, 128, 64, device=gpu)
    cache.export(c, arena)
    assert arena.layer_seq_lens == [54, 54]
    for layer in range(layers):
        keys, values = arena.attended(layer)
        assert torch.equal(keys, kept[id(c)][layer][0]) and torch.equal(values, kept[id(c)][layer][1])


def test_two_streams(gpu):
    """Appends to two layers on two streams."""
    cache = random_pool(gpu, 2, 8, 64, 64, seed=20)
    pools = [Pool(cache.storage[i], cache.exponents[i]) for i in range(2)]
    table, lens = tables(gpu, [list(range(32)), list(range(32, 64))]), ints(gpu, [2000, 1037])
    rows = [new_rows(2, 8, 40, seed=21 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    fed = [(k.to(gpu), v.to(gpu)) for k, v in rows]
    torch.cuda.synchronize()
    for i, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            kernels.paged_append(cache, i, *fed[i], table, lens)
    torch.cuda.synchronize()
    for i in range(2):
        pools[i].append(*rows[i], table.tolist(), lens.tolist())
        same(cache, pools[i], i)
