"""The low-rank adapters that a server keeps beside one shared projection.

An adapter of a projection W[N, K] is A [r, K] and B [N, r] with a scale; a row x
that names it gets scale * (x . A^T) . B^T added (kernels.lora_add,
kernels.lora_linear).  A store holds `count` of them in fixed slots on the GPU,
in the tiles that the kernels read, so that an adapter can be replaced between
calls (and between replays of a captured graph) without moving anything.  The
reference has no adapters.
"""

from __future__ import annotations

import torch

from . import _lib
from .layout import TILE_K, TILE_ROWS, check_shape

# 16-row tiles of the rank that the kernels are built for: ranks up to 16, 32, 48, 64, 96, 128.
RANK_TILES = (1, 2, 3, 4, 6, 8)
MAX_RANK = TILE_ROWS * RANK_TILES[-1]


def _pack_a(a: torch.Tensor) -> torch.Tensor:
    """A [..., R, K] (R a multiple of 16) in LAYOUT_MFMA16X32 (layout.pack_tensor), adapter by adapter."""
    *lead, r, k = a.shape
    return a.reshape(-1, r // TILE_ROWS, TILE_ROWS, k // TILE_K, 4, 8).permute(0, 1, 3, 4, 2, 5).reshape(*lead, -1)


def _pack_b(b: torch.Tensor, gate_up: bool) -> torch.Tensor:
    """B [..., N, R] (R a multiple of 16; [gate; up] rows for gate_up) as the
    tiles of lsk_lora_add_bf16: 32 columns x 16 ranks each (for gate_up of 32 gate
    rows, then of their up rows), a lane's 16 bytes from two rows 4 apart."""
    *lead, n, r = b.shape
    parts = 2 if gate_up else 1
    b = b.reshape(-1, parts, n // parts, r)
    rest = -(n // parts) % 32
    if rest:
        b = torch.cat((b, b.new_zeros(*b.shape[:2], rest, r)), 2)
    # row 32 j + 8 q + 4 half + i, rank 16 t + 4 g + e -> [j, t, part, g, (q, i), half, e]
    blocks = b.view(b.shape[0], parts, -1, 4, 2, 4, r // 16, 4, 4)
    return blocks.permute(0, 2, 6, 1, 7, 3, 5, 4, 8).reshape(*lead, -1)


class AdapterStore:
    """`count` adapters of rank up to `rank` for projections of [n, k] weights,
    all empty (they add nothing) until loaded.  gate_up: the projection is a
    fused [gate; up] one, whose SiLU(gate) * up is taken after the adapters.  A
    store holds values: of adapters that require gradients, no graph."""

    def __init__(self, count: int, n: int, k: int, rank: int, *, gate_up: bool = False,
                 device: torch.device | str = "cuda") -> None:
        check_shape(n, k, _lib.LAYOUT_MFMA16X32_GATEUP if gate_up else _lib.LAYOUT_MFMA16X32)
        if count < 1 or not 1 <= rank <= MAX_RANK:
            raise ValueError(f"a store needs at least one adapter and a rank of 1..{MAX_RANK}, got count={count}, "
                             f"rank={rank}")
        self.count, self.n, self.k, self.gate_up = count, n, k, gate_up
        self.rank_tiles = next(t for t in RANK_TILES if t * TILE_ROWS >= rank)
        self.rank = self.rank_tiles * TILE_ROWS
        self.a_tiles = torch.zeros((count, self.rank * k), device=device, dtype=torch.bfloat16)
        columns = -(-n // 64) * 64 if gate_up else -(-n // 32) * 32
        self.b_tiles = torch.zeros((count, columns * self.rank), device=device, dtype=torch.bfloat16)
        self.scales = torch.zeros((count,), device=device, dtype=torch.float32)
        self.ranks = torch.zeros((count,), device=device, dtype=torch.int32)

    @property
    def device(self) -> torch.device:
        return self.a_tiles.device

    @torch.no_grad()
    def load(self, slot: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """Put A [r, k] and B [n, r] (bfloat16, r up to the store's rank; a
        gate_up B's gate rows first) into a slot, on the current stream."""
        if not 0 <= slot < self.count:
            raise ValueError(f"slot {slot} is not one of the store's {self.count}")
        r = a.shape[0] if a.dim() == 2 else -1
        if a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16 or tuple(a.shape) != (r, self.k) \
                or tuple(b.shape) != (self.n, r) or not 1 <= r <= self.rank:
            raise ValueError(f"an adapter must be bfloat16 A [r, {self.k}] and B [{self.n}, r] with r of 1..{self.rank}, "
                             f"got {a.dtype} {tuple(a.shape)} and {b.dtype} {tuple(b.shape)}")
        rows = torch.zeros((self.rank, self.k), device=self.device, dtype=torch.bfloat16)
        cols = torch.zeros((self.n, self.rank), device=self.device, dtype=torch.bfloat16)
        rows[:r].copy_(a)
        cols[:, :r].copy_(b)
        self.a_tiles[slot].copy_(_pack_a(rows))
        self.b_tiles[slot].copy_(_pack_b(cols, self.gate_up))
        self.scales[slot:slot + 1].fill_(scale)
        self.ranks[slot:slot + 1].fill_(r)

    @torch.no_grad()
    def load_parts(self, slot: int, parts: list[tuple[torch.Tensor, torch.Tensor]], scale: float = 1.0) -> None:
        """One adapter per part of a fused projection ((A, B) of q, k and v, or
        of gate and up, in the order of the fused rows): their ranks stand
        beside each other, each part's B in its own rows."""
        if not parts:
            raise ValueError("an adapter needs at least one part")
        a = torch.cat([pa for pa, _ in parts]).to(self.device)
        self.load(slot, a, torch.block_diag(*(pb for _, pb in parts)).to(device=self.device, dtype=a.dtype), scale)

    @torch.no_grad()
    def clear(self, slot: int) -> None:
        """Empty a slot: rows that name it get nothing added."""
        if not 0 <= slot < self.count:
            raise ValueError(f"slot {slot} is not one of the store's {self.count}")
        self.b_tiles[slot].zero_()
        self.ranks[slot:slot + 1].fill_(0)

    @classmethod
    @torch.no_grad()
    def of(cls, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor, *, gate_up: bool = False) -> "AdapterStore":
        """A store of adapters held as A [count, r, k] and B [count, n, r] with scales [count]."""
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2] \
                or tuple(scales.shape) != (a.shape[0],) or a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16:
            raise ValueError(f"adapters must be bfloat16 A [count, r, k] and B [count, n, r] and scales [count], got "
                             f"{a.dtype} {tuple(a.shape)}, {b.dtype} {tuple(b.shape)} and {tuple(scales.shape)}")
        store = cls(a.shape[0], b.shape[1], a.shape[2], a.shape[1], gate_up=gate_up, device=a.device)
        rest = store.rank - a.shape[1]
        store.a_tiles.copy_(_pack_a(torch.nn.functional.pad(a, (0, 0, 0, rest))))
        store.b_tiles.copy_(_pack_b(torch.nn.functional.pad(b, (0, rest)), gate_up))
        store.scales.copy_(scales)
        store.ranks.fill_(a.shape[1])
        return store
