"""Constrained logits: what the wrapper and the C entry point refuse before
anything touches the device, and the slices that the vocabulary is cut into."""

from __future__ import annotations

import pytest
import torch

from leanstack_amd import _lib, kernels

FAKE = 0x10000  # aligned, never dereferenced
INVALID, WORKSPACE = -1, -4


@pytest.mark.parametrize("bad,code", [
    (dict(mode=2), INVALID), (dict(m=0), INVALID), (dict(v=0), INVALID), (dict(v=(1 << 30) + 1), INVALID),
    (dict(m=1 << 23), INVALID), (dict(ld=999), INVALID), (dict(logits=0), INVALID), (dict(out=0), INVALID),
    (dict(tokens=0), INVALID), (dict(logits=FAKE + 2), INVALID), (dict(out=FAKE + 2), INVALID),
    (dict(tokens=FAKE + 4), INVALID), (dict(out=FAKE, ld=1008), INVALID), (dict(history_len=0), INVALID),
    (dict(history_len=(1 << 20) + 1, history_ld=1 << 21), INVALID), (dict(history_ld=49), INVALID),
    (dict(history=FAKE + 2), INVALID), (dict(history=None), INVALID),
    (dict(history=None, lens=None, prompt=None, rep=None, freq=None), INVALID), (dict(rep=FAKE + 1), INVALID),
    (dict(nb=-1), INVALID), (dict(nb=1024, bias_ld=1024), INVALID), (dict(ids=None), INVALID), (dict(vals=None), INVALID),
    (dict(bias_ld=6), INVALID), (dict(allowed_ld=31), INVALID), (dict(allowed=FAKE + 2), INVALID),
    (dict(ws=None), WORKSPACE), (dict(ws=FAKE + 4), WORKSPACE), (dict(ws_bytes=8), WORKSPACE),
])
def test_entry_point_rejects_before_launch(bad, code):
    lib = _lib.load()
    a = dict(logits=FAKE, mode=0, m=3, v=1000, ld=1000, history=FAKE, history_ld=50, history_len=50, lens=FAKE,
             prompt=FAKE, rep=FAKE, freq=FAKE, pres=FAKE, ids=FAKE, vals=FAKE, bias_ld=7, nb=7, allowed=FAKE, allowed_ld=32,
             out=FAKE + 0x100000, tokens=FAKE, ws=FAKE) | bad
    if "ws_bytes" not in a:
        a["ws_bytes"] = lib.lsk_constrain_workspace_bytes(3, 1000)
    status = lib.lsk_constrain_logits(
        a["logits"], a["mode"], a["m"], a["v"], a["ld"], a["history"], a["history_ld"], a["history_len"], a["lens"],
        a["prompt"], a["rep"], a["freq"], a["pres"], a["ids"], a["vals"], a["bias_ld"], a["nb"], a["allowed"],
        a["allowed_ld"], a["out"], a["tokens"], a["ws"], a["ws_bytes"], None)
    assert status == code
    assert lib.lsk_last_error()


def test_workspace_bytes():
    """A counter of 64 bytes per row and a key of 8 per slice, slices of at most 10176 values."""
    lib = _lib.load()
    for m in (1, 2, 7, 64, 511, 512, 513, 4096):
        for v in (1, 63, 64, 65, 2048, 2049, 10176, 16321, 50257, 151936, 1 << 20, 1 << 30):
            slices, rest = divmod(lib.lsk_constrain_workspace_bytes(m, v) // m - 64, 8)
            assert rest == 0 and slices * 10176 >= v and slices <= max(v // 2048 + 1, -(-v // 10176) + 1)
    assert lib.lsk_constrain_workspace_bytes(0, 5) == 0 and lib.lsk_constrain_workspace_bytes(5, 0) == 0


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("kw,what", [
    (dict(history=_i(3, 5).long()), "history"), (dict(history=_i(2, 5)), "history"), (dict(history=_i(3)), "history"),
    (dict(history=_i(1, 5).expand(3, 5)), "repeat"), (dict(history=_i(5, 3).t()), "contiguous rows"),
    (dict(history=_i(1, 1 << 21).expand(3, -1)[:, : (1 << 20) + 1]), "repeat"),
    (dict(history=_i(3, 5), history_lens=_i(2)), "history_lens"), (dict(history=_i(3, 5), prompt_lens=_i(3).long()), "prompt"),
    (dict(history=_i(3, 5), repetition=torch.ones(3).double()), "repetition"), (dict(history_lens=_i(3)), "without a history"),
    (dict(presence=torch.ones(3)), "without a history"), (dict(bias_ids=_i(3, 2)), "go together"),
    (dict(bias_ids=_i(3, 2), bias_values=torch.ones(3, 3)), "strides"),
    (dict(bias_ids=_i(3, 1024), bias_values=torch.ones(3, 1024)), "1024 biases"),
    (dict(allowed=_i(3, 3)), "words"), (dict(allowed=_i(3, 4).long()), "allowed"), (dict(out=torch.ones(3, 99)), "out"),
    (dict(out=torch.ones(3, 100).bfloat16()), "out"), (dict(), "GPU"),
])
def test_wrapper_refuses(kw, what):
    with pytest.raises(ValueError, match=what):
        kernels.constrain_logits(torch.ones(3, 100), **kw)


def test_wrapper_refuses_logits():
    for bad in (torch.ones(3, 100).half(), torch.ones(300), torch.ones(3, 0)):
        with pytest.raises(ValueError, match="logits"):
            kernels.constrain_logits(bad)
    room = torch.ones(400)
    with pytest.raises(ValueError, match="overlap"):
        kernels.constrain_logits(room[:300].view(3, 100), out=room[50:350].view(3, 100))
