"""Low-rank adapters: the packed layout of a store, what the wrappers and the C
entry point refuse before anything touches the device, and the plan's sizes."""

from __future__ import annotations

import pytest
import torch

from leanstack_amd import _lib, kernels
from leanstack_amd.adapters import RANK_TILES, AdapterStore, _pack_b
from leanstack_amd.layout import PackedWeight, unpack_tensor
from tests.helpers import seeded_normal

FAKE = 0x10000  # aligned, never dereferenced
INVALID, WORKSPACE = -1, -4


@pytest.mark.parametrize("n,r,gate_up", [(32, 16, False), (48, 32, False), (16, 16, False), (192, 64, True), (96, 16, True)])
def test_b_tiles_follow_the_documented_layout(n, r, gate_up):
    b = seeded_normal((n, r), 1.0, n + r)
    parts = 2 if gate_up else 1
    tiles = _pack_b(b, gate_up).view(-1, r // 16, parts, 64, 8)  # [columns, rank tile, part, lane, value]
    assert tiles.shape[0] == (n // parts + 31) // 32
    for j in range(tiles.shape[0]):
        for t in range(r // 16):
            for p in range(parts):
                for lane in range(64):
                    g, c = lane // 16, lane % 16
                    for e in range(4):
                        for half in range(2):
                            row = 32 * j + 8 * (c // 4) + c % 4 + 4 * half
                            want = float(b[p * n // 2 + row, 16 * t + 4 * g + e]) if row < n // parts else 0.0
                            assert float(tiles[j, t, p, lane, 4 * half + e]) == want
    store = AdapterStore(1, n, 32, r, gate_up=gate_up, device="cpu")
    assert store.b_tiles[0].numel() == tiles.numel()


def test_a_store_holds_what_is_loaded():
    store = AdapterStore(2, 48, 64, 20, device="cpu")
    assert store.rank == 32 and store.rank_tiles == 2
    a, b = seeded_normal((20, 64), 1.0, 1), seeded_normal((48, 20), 1.0, 2)
    store.load(1, a, b, 0.5)
    rows = unpack_tensor(store.a_tiles[1], 32, 64)
    assert torch.equal(rows[:20], a) and not bool(rows[20:].any())
    assert store.ranks.tolist() == [0, 20] and store.scales.tolist() == [0.0, 0.5]
    store.clear(1)
    assert store.ranks.tolist() == [0, 0]
    for bad in ((2, a, b), (-1, a, b), (0, a.float(), b), (0, a, b.float()), (0, a[:, :32], b), (0, a, b[:32]),
                (0, a[:19], b), (0, a[:0], b[:, :0]), (0, seeded_normal((33, 64), 1, 1), seeded_normal((48, 33), 1, 1)),
                (0, a[0], b)):
        with pytest.raises(ValueError):
            store.load(*bad)
    for bad in (2, -1):
        with pytest.raises(ValueError):
            store.clear(bad)
    with pytest.raises(ValueError):
        store.load_parts(0, [])
    for bad in (dict(count=0), dict(rank=0), dict(rank=129), dict(n=40), dict(k=40), dict(n=48, gate_up=True)):
        with pytest.raises(ValueError):
            AdapterStore(**(dict(count=1, n=64, k=64, rank=8, device="cpu") | bad))
    with pytest.raises(ValueError):
        AdapterStore.of(torch.zeros(2, 4, 64), torch.zeros(3, 48, 4), torch.zeros(2))


@pytest.mark.parametrize("bad,code", [
    (dict(m=0), INVALID), (dict(n=40), INVALID), (dict(k=40), INVALID), (dict(n=48, ldy=48, epi=1), INVALID),
    (dict(epi=2), INVALID), (dict(epi=7), INVALID), (dict(count=0), INVALID), (dict(rt=0), INVALID), (dict(rt=5), INVALID),
    (dict(rt=9), INVALID), (dict(ldx=9720), INVALID), (dict(ldx=9732), INVALID), (dict(ldx=1 << 22), INVALID),
    (dict(ldy=2552), INVALID), (dict(ldy=2564), INVALID), (dict(y=0), INVALID), (dict(x=FAKE + 8), INVALID),
    (dict(a=0), INVALID), (dict(b=FAKE + 8), INVALID), (dict(out=FAKE + 8), INVALID), (dict(scale=0), INVALID),
    (dict(ranks=FAKE + 2), INVALID), (dict(index=None), INVALID), (dict(out=FAKE, ldy=2568), INVALID),
    (dict(out=FAKE, epi=1), INVALID), (dict(m=0x7fffffff), INVALID), (dict(ws=None), WORKSPACE),
    (dict(ws=FAKE + 8), WORKSPACE), (dict(ws_bytes=16), WORKSPACE),
])
def test_entry_point_rejects_before_launch(bad, code):
    lib = _lib.load()
    a = dict(y=FAKE, m=20, n=2560, ldy=2560, x=FAKE, k=9728, ldx=9728, a=FAKE, b=FAKE, scale=FAKE, ranks=FAKE, count=6,
             rt=4, index=FAKE, epi=0, out=FAKE + 0x100000, ws=FAKE) | bad
    need = lib.lsk_lora_workspace_bytes(20, 2560, 9728, 4, 6, 0)
    assert need > 0
    a.setdefault("ws_bytes", need)
    status = lib.lsk_lora_add_bf16(a["y"], a["m"], a["n"], a["ldy"], a["x"], a["k"], a["ldx"], a["a"], a["b"], a["scale"],
                                   a["ranks"], a["count"], a["rt"], a["index"], a["epi"], a["out"], a["ws"],
                                   a["ws_bytes"], None)
    assert status == code
    assert lib.lsk_last_error()


def test_workspace_bytes():
    """Whole fp32 partials of h, at most 8; 64 rows to a tile above 128 rows."""
    lib = _lib.load()
    for m in (1, 16, 17, 128, 129, 300, 5000):
        for n, k in ((16, 32), (2560, 9728), (19456, 2560)):
            for rt in RANK_TILES:
                rows = 16 if m <= 128 else 64
                tile = -(-m // rows) * rows * rt * 64
                splits, rest = divmod(lib.lsk_lora_workspace_bytes(m, n, k, rt, 5, 0), tile)
                assert rest == 0 and splits <= 8 and (m <= 128 or splits >= 1)
    for bad in ((0, 16, 32, 1, 1), (1, 0, 32, 1, 1), (1, 16, 0, 1, 1), (1, 16, 32, 5, 1), (1, 16, 32, 1, 0)):
        assert lib.lsk_lora_workspace_bytes(*bad, 0) == 0


def test_wrappers_refuse():
    store = AdapterStore(2, 64, 32, 8, device="cpu")
    gate_up = AdapterStore(2, 64, 32, 8, gate_up=True, device="cpu")
    y, x, index = seeded_normal((3, 64), 1, 1), seeded_normal((3, 32), 1, 2), torch.zeros(3, dtype=torch.int32)
    weight = PackedWeight.from_rowmajor(seeded_normal((64, 32), 1, 3))
    gu = PackedWeight.from_rowmajor(seeded_normal((64, 32), 1, 3), _lib.LAYOUT_MFMA16X32_GATEUP)
    for args, kw, what in [
        ((y, x, (1, 2), index), {}, "AdapterStore"), ((y.float(), x, store, index), {}, "bfloat16"),
        ((y[:, :32], x, store, index), {}, "last dim"), ((y, x[:2], store, index), {}, "rows"),
        ((y, x, store, index.long()), {}, "index"), ((y, x, store, index[:2]), {}, "index"),
        ((y, x, store, index), {"epilogue": 1}, "epilogue"), ((y, x, gate_up, index), {}, "epilogue"),
        ((y, x, store, index), {"epilogue": 2}, "epilogue"), ((y, x, store, index), {"out": y[:2]}, "out"),
        ((y, x, store, index), {"out": y.float()}, "out"), ((y, x, gate_up, index), {"epilogue": 1, "out": y[:, :32]}, "out"),
        ((y, x, store, index), {}, "GPU"),
    ]:
        with pytest.raises(ValueError, match=what):
            kernels.lora_add(*args, **kw)
    room = torch.zeros(3 * 64 + 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):
        kernels.lora_add(room[:192].view(3, 64), x, store, index, out=room[64:].view(3, 64))
    for args, kw, what in [
        ((x, y, store, index), {}, "PackedWeight"), ((x, weight, gate_up, index), {}, "gate_up"),
        ((x, gu, gate_up, index), {}, "gate_up"), ((x, gu, store, index), {"epilogue": 1}, "gate_up"),
        ((x, PackedWeight.from_rowmajor(seeded_normal((32, 32), 1, 3)), store, index), {}, "shape"),
        ((x, gu, gate_up, index), {"epilogue": 1, "residual": y}, "residual"),
    ]:
        with pytest.raises(ValueError, match=what):
            kernels.lora_linear(*args, **kw)
