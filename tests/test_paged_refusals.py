"""The paged 8-bit cache: what the wrappers and the C entry points refuse before anything touches the device."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from leanstack_amd import _lib, kernels
from leanstack_amd.paged_cache import PagedKVCache

FAKE = 0x10000  # aligned, never dereferenced
INVALID, WORKSPACE = -1, -4
POOL = dict(k=FAKE, v=FAKE, ke=FAKE, ve=FAKE, pages=100, n_kv=8, page_rows=64, table_pages=20, table=FAKE, stride=20)

BAD_POOLS = [dict(page_rows=48), dict(page_rows=8), dict(page_rows=2048), dict(page_rows=0), dict(page_rows=-16), dict(pages=0),
             dict(pages=-1), dict(n_kv=0), dict(table_pages=0), dict(stride=19), dict(k=None), dict(v=None), dict(k=FAKE + 8),
             dict(v=FAKE + 1), dict(ke=None), dict(ve=None), dict(table=None), dict(table=FAKE + 2), dict(pages=1 << 30),
             dict(n_kv=1 << 30), dict(table_pages=1 << 25, stride=1 << 25)]


def pool_of(a):
    p = POOL | {key: a[key] for key in POOL if key in a}
    return _lib.PagedPool(p["k"], p["v"], p["ke"], p["ve"], p["pages"], p["n_kv"], p["page_rows"], p["table_pages"], p["table"],
                          p["stride"])


def refused(status, code):
    assert status == code
    assert _lib.load().lsk_last_error()


@pytest.mark.parametrize("bad", BAD_POOLS + [
    dict(b=0), dict(t=0), dict(t=-1), dict(b=1 << 22, t=1 << 22), dict(t=(1 << 31) - 1), dict(kb=4), dict(kh=-8), dict(kt=12),
    dict(vb=-8), dict(vh=1), dict(vt=4), dict(x=None), dict(x=FAKE + 8), dict(y=None), dict(y=FAKE + 2), dict(lens=None),
    dict(lens=FAKE + 1), dict(counts=FAKE + 2)])
def test_append_rejects_before_launch(bad):
    a = dict(x=FAKE, kb=1024, kh=128, kt=128, y=FAKE, vb=1024, vh=128, vt=128, b=3, t=5, lens=FAKE, counts=None) | bad
    refused(_lib.load().lsk_paged_append_bf16(ctypes.byref(pool_of(bad)), a["x"], a["kb"], a["kh"], a["kt"], a["y"], a["vb"],
                                              a["vh"], a["vt"], a["b"], a["t"], a["lens"], a["counts"], None), INVALID)


@pytest.mark.parametrize("bad", BAD_POOLS + [
    dict(b=0), dict(rows=0), dict(rows=-5), dict(b=1 << 22, rows=1 << 22), dict(starts=None), dict(starts=FAKE + 2),
    dict(lens=FAKE + 1), dict(x=None), dict(x=FAKE + 8), dict(y=None), dict(y=FAKE + 4)])
def test_read_rejects_before_launch(bad):
    a = dict(starts=FAKE, lens=None, b=3, rows=40, x=FAKE, y=FAKE) | bad
    refused(_lib.load().lsk_paged_read_bf16(ctypes.byref(pool_of(bad)), a["starts"], a["lens"], a["b"], a["rows"], a["x"],
                                            a["y"], None), INVALID)


@pytest.mark.parametrize("bad", [
    dict(storage=None), dict(storage=FAKE + 8), dict(exponents=None), dict(planes=0), dict(pages=0), dict(blocks=0),
    dict(blocks=(1 << 20) + 1), dict(src=None), dict(src=FAKE + 2), dict(dst=None), dict(dst=FAKE + 1), dict(n=0), dict(n=-1),
    dict(n=1 << 30, planes=72), dict(n=1 << 20, planes=72, blocks=1 << 10)])
def test_copy_rejects_before_launch(bad):
    a = dict(storage=FAKE, exponents=FAKE, planes=72, pages=50, blocks=32, src=FAKE, dst=FAKE, n=3) | bad
    refused(_lib.load().lsk_paged_copy(a["storage"], a["exponents"], a["planes"], a["pages"], a["blocks"], a["src"], a["dst"],
                                       a["n"], None), INVALID)


@pytest.mark.parametrize("bad,code", [(bad, INVALID) for bad in BAD_POOLS] + [
    (dict(d=64), INVALID), (dict(n_q=30), INVALID), (dict(n_q=4), INVALID), (dict(n_q=0), INVALID), (dict(b=0), INVALID),
    (dict(t=0), INVALID), (dict(b=1 << 20, t=1 << 10), INVALID), (dict(qb=-8), INVALID), (dict(qh=4), INVALID),
    (dict(qt=2), INVALID), (dict(q=None), INVALID), (dict(q=FAKE + 8), INVALID), (dict(lens=None), INVALID),
    (dict(lens=FAKE + 2), INVALID), (dict(counts=FAKE + 1), INVALID), (dict(out=None), INVALID), (dict(out=FAKE + 8), INVALID),
    (dict(scale=math.nan), INVALID), (dict(scale=math.inf), INVALID), (dict(scale=-1e37), INVALID)])
def test_attention_rejects_before_launch(bad, code):
    lib = _lib.load()
    a = dict(q=FAKE, qb=4096, qh=128, qt=4096, b=3, t=2, n_q=32, d=128, lens=FAKE, counts=None, scale=0.1, out=FAKE, ws=FAKE,
             ws_bytes=1 << 40) | bad
    refused(lib.lsk_paged_attention_bf16(ctypes.byref(pool_of(bad)), a["q"], a["qb"], a["qh"], a["qt"], a["b"], a["t"], a["n_q"],
                                         a["d"], a["lens"], a["counts"], a["scale"], a["out"], a["ws"], a["ws_bytes"], None), code)


def test_a_null_pool_is_refused():
    lib = _lib.load()
    refused(lib.lsk_paged_append_bf16(None, FAKE, 8, 8, 8, FAKE, 8, 8, 8, 1, 1, FAKE, None, None), INVALID)
    refused(lib.lsk_paged_read_bf16(None, FAKE, None, 1, 1, FAKE, FAKE, None), INVALID)
    refused(lib.lsk_paged_attention_bf16(None, FAKE, 8, 8, 8, 1, 1, 8, 128, FAKE, None, 0.1, FAKE, None, 0, None), INVALID)


def cache_and_rows(b=2, t=3, n_kv=2):
    cache = PagedKVCache(2, n_kv, 6, page_rows=16)
    k = torch.zeros((b, n_kv, t, 128), dtype=torch.bfloat16)
    return cache, k, torch.zeros((b, 2), dtype=torch.int32), torch.zeros(b, dtype=torch.int32)


def test_wrappers_refuse():
    cache, k, table, lens = cache_and_rows()
    q = torch.zeros((2, 4, 3, 128), dtype=torch.bfloat16)
    calls = [
        lambda: kernels.paged_append(None, 0, k, k, table, lens),
        lambda: kernels.paged_append(cache, 2, k, k, table, lens),
        lambda: kernels.paged_append(cache, -1, k, k, table, lens),
        lambda: kernels.paged_append(cache, 0, k.float(), k, table, lens),
        lambda: kernels.paged_append(cache, 0, k[:, :1], k[:, :1], table, lens),
        lambda: kernels.paged_append(cache, 0, k, k[:, :, :2], table, lens),
        lambda: kernels.paged_append(cache, 0, k[..., :64], k[..., :64], table, lens),
        lambda: kernels.paged_append(cache, 0, k[:1], k[:1], table, lens),
        lambda: kernels.paged_append(cache, 0, k, k, table.long(), lens),
        lambda: kernels.paged_append(cache, 0, k, k, table[0], lens),
        lambda: kernels.paged_append(cache, 0, k, k, table[:1].expand(2, 2), lens),
        lambda: kernels.paged_append(cache, 0, k, k, table.t(), lens),
        lambda: kernels.paged_append(cache, 0, k, k, table, lens.long()),
        lambda: kernels.paged_append(cache, 0, k, k, table, lens[:1]),
        lambda: kernels.paged_append(cache, 0, k, k, table, lens, counts=lens[:1]),
        lambda: kernels.paged_append(cache, 0, k, k, table, None),
        lambda: kernels.paged_append(cache, 0, k, k, table, lens),  # not on a GPU
        lambda: kernels.paged_read(cache, 0, table, lens, -1),
        lambda: kernels.paged_read(cache, 0, table, lens[:1], 4),
        lambda: kernels.paged_read(cache, 0, table, lens, 4),
        lambda: kernels.copy_pages(cache, lens, lens[:1]),
        lambda: kernels.copy_pages(cache, lens.long(), lens.long()),
        lambda: kernels.copy_pages(None, lens, lens),
        lambda: kernels.copy_pages(cache, lens, lens),
        lambda: kernels.paged_attention(q.float(), cache, 0, table, lens, 0.1),
        lambda: kernels.paged_attention(q[:, :3], cache, 0, table, lens, 0.1),
        lambda: kernels.paged_attention(q[:1], cache, 0, table, lens, 0.1),
        lambda: kernels.paged_attention(q[..., :64], cache, 0, table, lens, 0.1),
        lambda: kernels.paged_attention(q, cache, 0, table, lens, 0.1, counts=lens.long()),
        lambda: kernels.paged_attention(q, cache, 0, table, lens, 0.1, out=q),
        lambda: kernels.paged_attention(q, cache, 0, table, lens, 0.1, out=torch.zeros((2, 3, 512))),
        lambda: kernels.paged_attention(q, cache, 0, table, lens, 0.1),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
