"""Attention over a shared prefix: what the wrapper and the C entry point refuse
before anything touches the device, and the workspace's size."""

from __future__ import annotations

import math

import pytest
import torch

from leanstack_amd import _lib, kernels

FAKE = 0x10000  # aligned, never dereferenced
INVALID, WORKSPACE = -1, -4


@pytest.mark.parametrize("bad,code", [
    (dict(d=64), INVALID), (dict(n_kv=0), INVALID), (dict(n_q=30), INVALID), (dict(n_q=4), INVALID), (dict(b=0), INVALID),
    (dict(t=0), INVALID), (dict(p=-1), INVALID), (dict(s=-1), INVALID), (dict(b=1 << 20, t=1 << 10), INVALID),
    (dict(b=1 << 19, s=1 << 20), INVALID), (dict(p_row=120), INVALID), (dict(p_row=132), INVALID), (dict(row=64), INVALID),
    (dict(row=132), INVALID), (dict(p=1 << 23), INVALID), (dict(s=1 << 23), INVALID), (dict(p=1 << 20, p_row=1024), INVALID),
    (dict(p_row=1 << 22), INVALID), (dict(row=1 << 22), INVALID),
    (dict(q_b=-8), INVALID), (dict(q_h=4), INVALID), (dict(q_t=12), INVALID), (dict(p_head=-8), INVALID),
    (dict(batch=4), INVALID), (dict(head=2), INVALID), (dict(q=0), INVALID), (dict(q=FAKE + 8), INVALID), (dict(pk=0), INVALID),
    (dict(pv=FAKE + 8), INVALID), (dict(k=0), INVALID), (dict(v=FAKE + 2), INVALID), (dict(lens=None), INVALID),
    (dict(lens=FAKE + 2), INVALID), (dict(out=0), INVALID), (dict(out=FAKE + 8), INVALID), (dict(scale=math.nan), INVALID),
    (dict(scale=math.inf), INVALID), (dict(ws=None), WORKSPACE), (dict(ws=FAKE + 8), WORKSPACE), (dict(ws_bytes=64), WORKSPACE),
])
def test_entry_point_rejects_before_launch(bad, code):
    lib = _lib.load()
    a = dict(q=FAKE, q_b=4096, q_h=128, q_t=4096, b=5, t=2, n_q=32, n_kv=8, d=128, pk=FAKE, pv=FAKE, p_head=128 * 1000,
             p_row=128, p=1000, k=FAKE, v=FAKE, batch=8 * 128 * 400, head=128 * 400, row=128, s=400, lens=FAKE, scale=0.1,
             out=FAKE, ws=FAKE) | bad
    need = lib.lsk_prefix_attention_workspace_bytes(5, 2, 32, 8, 1000, 400)
    assert need > 0
    a.setdefault("ws_bytes", need)
    status = lib.lsk_prefix_attention_bf16(
        a["q"], a["q_b"], a["q_h"], a["q_t"], a["b"], a["t"], a["n_q"], a["n_kv"], a["d"], a["pk"], a["pv"], a["p_head"],
        a["p_row"], a["p"], a["k"], a["v"], a["batch"], a["head"], a["row"], a["s"], a["lens"], a["scale"], a["out"], a["ws"],
        a["ws_bytes"], None)
    assert status == code
    assert lib.lsk_last_error()


def test_workspace_bytes():
    """Whole parts of 130 fp32 values per query row; none for short contexts and bad shapes."""
    bytes_of = _lib.load().lsk_prefix_attention_workspace_bytes
    for b, t, n_q, n_kv in ((1, 1, 32, 8), (64, 1, 32, 8), (3, 16, 8, 1), (200, 4, 16, 16)):
        for p, s in ((0, 1000), (1000, 0), (5000, 300), (16384, 1088), (100000, 1)):
            nbytes = bytes_of(b, t, n_q, n_kv, p, s)
            assert nbytes > 0 and nbytes % (b * t * n_q * 130 * 4) == 0
    assert bytes_of(4, 1, 32, 8, 0, 0) == 0 and bytes_of(4, 1, 32, 8, 64, 30) == 0
    for bad in ((0, 1, 8, 8, 999, 9), (1, 0, 8, 8, 999, 9), (1, 1, 8, 0, 999, 9), (1, 1, 9, 8, 999, 9), (1, 1, 8, 8, -1, 9),
                (1, 1, 8, 8, 999, -1)):
        assert bytes_of(*bad) == 0


def _bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("bad,what", [
    (dict(q=_bf(3, 8, 128)), "must be"), (dict(q=_bf(3, 8, 2, 128).float()), "q must be bfloat16"),
    (dict(q=_bf(3, 8, 2, 64)), "fit"), (dict(q=_bf(3, 7, 2, 128)), "fit"), (dict(q=_bf(2, 8, 2, 128)), "fit"),
    (dict(prefix_k=_bf(4, 10, 128)), "fit"), (dict(prefix_v=_bf(2, 11, 128)), "one shape"),
    (dict(prefix_k=_bf(2, 10, 128).float()), "bfloat16"), (dict(k=_bf(3, 4, 5, 128)), "fit"),
    (dict(v=_bf(3, 2, 5, 128).half()), "bfloat16"), (dict(v=_bf(3, 5, 2, 128).transpose(1, 2)), "strides"),
    (dict(k=_bf(3, 2, 5, 256)[..., ::2], v=_bf(3, 2, 5, 256)[..., ::2]), "strides"),
    (dict(k=_bf(3, 2, 5, 132)[..., :128], v=_bf(3, 2, 5, 132)[..., :128]), "strides"),
    (dict(k=_bf(3, 2, 1, 128).expand(-1, -1, 5, -1), v=_bf(3, 2, 1, 128).expand(-1, -1, 5, -1)), "repeat"),
    (dict(lens=torch.zeros(3)), "lens"), (dict(lens=torch.zeros(2, dtype=torch.int32)), "lens"),
    (dict(lens=torch.zeros(3, dtype=torch.int64)), "lens"), (dict(out=_bf(3, 2, 8, 128)), "out"),
    (dict(out=_bf(3, 2, 1024).float()), "out"), (dict(), "GPU"),
])
def test_wrapper_refuses(bad, what):
    args = dict(q=_bf(3, 8, 2, 128), prefix_k=_bf(2, 10, 128), prefix_v=_bf(2, 10, 128), k=_bf(3, 2, 5, 128),
                v=_bf(3, 2, 5, 128), lens=torch.zeros(3, dtype=torch.int32), scale=0.1) | bad
    with pytest.raises(ValueError, match=what):
        kernels.shared_prefix_attention(**args)


def test_wrapper_refuses_an_output_over_its_inputs():
    q = _bf(3, 8, 2, 128)
    with pytest.raises(ValueError, match="overlap"):
        kernels.shared_prefix_attention(q, _bf(2, 10, 128), _bf(2, 10, 128), _bf(3, 2, 5, 128), _bf(3, 2, 5, 128),
                                        torch.zeros(3, dtype=torch.int32), 0.1, out=q.view(3, 2, 1024))
