"""Sampled tokens: what the wrapper and the C entry point refuse before anything touches the device."""

from __future__ import annotations

import pytest
import torch

from leanstack_amd import _lib, kernels

FAKE = 0x10000  # aligned, never dereferenced
INVALID, WORKSPACE = -1, -4


@pytest.mark.parametrize("bad,code", [
    (dict(mode=2), INVALID), (dict(mode=-1), INVALID), (dict(m=0), INVALID), (dict(v=0), INVALID), (dict(v=(1 << 19) + 1), INVALID),
    (dict(m=1 << 23), INVALID), (dict(ld=999), INVALID), (dict(x=None), INVALID), (dict(x=FAKE + 2), INVALID),
    (dict(x=FAKE + 1, mode=1), INVALID), (dict(u=None), INVALID), (dict(u=FAKE + 2), INVALID), (dict(t=FAKE + 2), INVALID),
    (dict(k=FAKE + 1), INVALID), (dict(p=FAKE + 2), INVALID), (dict(mp=FAKE + 2), INVALID), (dict(tokens=None), INVALID),
    (dict(tokens=FAKE + 4), INVALID), (dict(logs=None), INVALID), (dict(logs=FAKE + 2), INVALID),
    (dict(v=50000, ld=50000, ws=None), WORKSPACE), (dict(v=50000, ld=50000, ws=FAKE + 8), WORKSPACE),
    (dict(v=50000, ld=50000, ws_bytes=100), WORKSPACE), (dict(v=50000, ld=50000, p=FAKE, ws_bytes=60000), WORKSPACE),
    (dict(v=1 << 19, ld=1 << 19, m=128, p=FAKE, ws_bytes=0), WORKSPACE),
])
def test_entry_point_rejects_before_launch(bad, code):
    lib = _lib.load()
    a = dict(x=FAKE, mode=0, m=3, v=1000, ld=1000, u=FAKE, t=None, k=None, p=None, mp=None, tokens=FAKE, logs=FAKE, ws=FAKE,
             ws_bytes=1 << 30) | bad
    status = lib.lsk_sample_logits(a["x"], a["mode"], a["m"], a["v"], a["ld"], a["u"], a["t"], a["k"], a["p"], a["mp"],
                                   a["tokens"], a["logs"], a["ws"], a["ws_bytes"], None)
    assert status == code
    assert lib.lsk_last_error()


def test_wrapper_refuses():
    x, u, k = torch.zeros((3, 40)), torch.zeros(3), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: kernels.sample_logits(x.half(), u), lambda: kernels.sample_logits(x[0], u), lambda: kernels.sample_logits(x[:, :0], u),
                 lambda: kernels.sample_logits(torch.zeros((1, (1 << 19) + 1)), u[:1]), lambda: kernels.sample_logits(x, u[:2]),
                 lambda: kernels.sample_logits(x, None), lambda: kernels.sample_logits(x, u.double()),
                 lambda: kernels.sample_logits(x, u, temperature=u[:1]), lambda: kernels.sample_logits(x, u, top_k=u),
                 lambda: kernels.sample_logits(x, u, top_k=k.long()), lambda: kernels.sample_logits(x, u, top_p=k),
                 lambda: kernels.sample_logits(x, u, min_p=u[:, None]), lambda: kernels.sample_logits(x, u)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("m,v,filters,some", [
    (1, 151936, (0, 0, 0), True), (1, 151936, (0, 1, 0), True), (170, 24576, (0, 1, 0), True), (1, 1 << 19, (0, 1, 0), True),
    (1, 151936, (1, 1, 0), True), (1, 151936, (0, 1, 1), True), (171, 151936, (0, 1, 0), False), (1, 24575, (0, 1, 0), False),
    (171, 151936, (1, 0, 0), False), (1, 65535, (1, 0, 1), False),
    (0, 151936, (0, 1, 0), False), (1, (1 << 19) + 1, (0, 0, 0), False),
])
def test_workspace_bytes(m, v, filters, some):
    """Only rows that are cut need one: with top-k or min-p 16 KB a slice, else 8 bytes of sums for 256 values, and with
    top-p 20 KB a slice."""
    need = [_lib.load().lsk_sample_workspace_bytes(mode, m, v, *filters) for mode in (0, 1)]
    assert (need[0] > 0) == some and need[1] in (need[0], 0)   # (bf16 rows are half as long)
    most = 16 * 16384 if filters[0] or filters[2] else v // 256 * 8 + (16 * 20480 if filters[1] else 0)
    assert need[0] <= m * (512 + most)
    assert _lib.load().lsk_sample_workspace_bytes(2, m, v, *filters) == 0
