"""A paged 8-bit cache from its definition (include/leanstack_amd.h), in 64 bits on the CPU."""

from __future__ import annotations

import math

import numpy as np
import torch

BLOCK, D = 16, 128
LEAST, MOST = -100, 119

# The finite e4m3 numbers that are not negative, by byte 0x00..0x7e: 4 exponent bits of bias 7, 3 fraction bits.
E4M3 = np.array([(b & 7) / 8 * 2.0 ** -6 if b < 8 else (1 + (b & 7) / 8) * 2.0 ** ((b >> 3) - 7) for b in range(0x7F)])


def places() -> tuple[np.ndarray, np.ndarray]:
    """Byte of (row, dim) in a block of keys and of values, [16, 128] each."""
    t, d = np.arange(BLOCK)[:, None], np.arange(D)[None]
    keys = d // 64 * 1024 + (d // 16 % 4 * 16 + t) * 16 + d % 16
    values = d // 16 % 2 * 1024 + (t // 4 * 16 + d % 16) * 16 + d // 32 * 4 + t % 4
    return keys, values


def nearest_byte(y: np.ndarray) -> np.ndarray:
    """The e4m3 byte nearest to y (|y| clipped to 448), ties to the even byte; NaN and infinities 0x7f."""
    fine = np.isfinite(y)
    size = np.minimum(np.abs(np.where(fine, y, 0.0)), 448.0)
    up = np.minimum(np.searchsorted(E4M3, size, "left"), 0x7E)
    down = np.maximum(up - 1, 0)
    below, above = size - E4M3[down], E4M3[up] - size
    byte = np.where(below < above, down, np.where(above < below, up, np.where(up % 2 == 0, up, down)))
    byte = byte.astype(np.uint8) | (np.signbit(y).astype(np.uint8) << 7)
    return np.where(fine, byte, 0x7F).astype(np.uint8)


def number(byte: np.ndarray) -> np.ndarray:
    size = np.append(E4M3, np.nan)[byte & 0x7F]
    return np.where(byte & 0x80, -size, size)


def least_exponent(x: np.ndarray) -> int:
    top = np.abs(x[np.isfinite(x)]).max(initial=0.0)
    e = LEAST
    while e < MOST and top > 448 * 2.0 ** e:
        e += 1
    return e


class Pool:
    """One layer's blocks and exponents, [2, pages, n_kv, blocks, ...], as numpy arrays."""

    def __init__(self, storage: torch.Tensor, exponents: torch.Tensor) -> None:
        self.bytes = storage.cpu().numpy().copy()
        self.exponents = exponents.cpu().numpy().copy()
        self.place = places()
        self.page_rows = self.bytes.shape[3] * BLOCK

    def numbers(self, kv: int, page: int, head: int, block: int) -> np.ndarray:
        """[16, 128] bytes of a block, by row and dim."""
        return self.bytes[kv, page, head, block][self.place[kv]]

    def append(self, k, v, table, lens, counts=None) -> None:
        """k / v [B, n_kv, T, D] (any tensors), table [B, P], lens, counts lists."""
        pages = self.bytes.shape[1]
        for b, n in enumerate(lens):
            count = k.shape[2] if counts is None else min(max(counts[b], 0), k.shape[2])
            start = max(n, 0) - count
            rows = [r for r in range(max(start, 0), max(n, 0)) if r < len(table[b]) * self.page_rows
                    and 0 <= table[b][r // self.page_rows] < pages]
            for block in sorted({r // BLOCK for r in rows}):
                mine = [r for r in rows if r // BLOCK == block]
                page, at = table[b][block * BLOCK // self.page_rows], block % (self.page_rows // BLOCK)
                for kv, x in enumerate((k, v)):
                    for head in range(x.shape[1]):
                        new = x[b, head, mine[0] - start:mine[-1] + 1 - start].double().numpy()
                        first = mine[0] - block * BLOCK
                        e = least_exponent(new)
                        byte = self.numbers(kv, page, head, at).copy()
                        if first:
                            was = int(self.exponents[kv, page, head, at]) - 127
                            e = max(e, was)
                            if e != was:
                                byte[:first] = nearest_byte(number(byte[:first]) * 2.0 ** (was - e))
                        byte[first:first + len(new)] = nearest_byte(new * 2.0 ** -e)
                        self.bytes[kv, page, head, at][self.place[kv]] = byte
                        self.exponents[kv, page, head, at] = e + 127

    def rows(self, kv: int, table_row, head: int, first: int, count: int) -> np.ndarray:
        """Values of a request's rows, float64 [count, D], and NaN-free zeros where there is no page."""
        out = np.zeros((count, D))
        for i in range(count):
            r = first + i
            if r < 0 or r >= len(table_row) * self.page_rows or not 0 <= table_row[r // self.page_rows] < self.bytes.shape[1]:
                continue
            page, at = table_row[r // self.page_rows], r % self.page_rows
            byte = self.bytes[kv, page, head, at // BLOCK][self.place[kv][at % BLOCK]]
            out[i] = number(byte) * 2.0 ** (int(self.exponents[kv, page, head, at // BLOCK]) - 127)
        return out

    def dense(self, table_row, rows: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """k, v float64 [n_kv, rows, D] of a request and which rows have a page, [rows]."""
        n_kv = self.bytes.shape[2]
        pages = np.array(table_row)[np.arange(rows) // self.page_rows] if rows else np.zeros(0, dtype=np.int64)
        there = (pages >= 0) & (pages < self.bytes.shape[1])
        pages = np.where(there, pages, 0)
        at = np.arange(rows) % self.page_rows
        both = []
        for kv in range(2):
            byte = self.bytes[kv][pages[:, None, None], np.arange(n_kv)[None, :, None], (at // BLOCK)[:, None, None],
                                  self.place[kv][at % BLOCK][:, None]]
            e = self.exponents[kv][pages[:, None], np.arange(n_kv)[None], (at // BLOCK)[:, None]].astype(np.float64) - 127
            x = number(byte) * 2.0 ** e[..., None]
            both.append(torch.from_numpy(np.where(there[:, None, None], x, 0.0)).transpose(0, 1).contiguous())
        return both[0], both[1], torch.from_numpy(there)


def attention(pool: Pool, q: torch.Tensor, table, lens, scale: float, counts=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(out, bound) float64 [B, T, n_q, D] of paged attention: the result, and how far a kernel may be that
    rounds as the entry point says it does.

    The bound, with h = 2^-8 the most that a rounding to bf16 is off, and p the weights: the output's own
    rounding, h |out|; the weights' roundings, each at most h and once more through the sum that divides, 2 h sum p |v|;
    the scores' errors, each at most 130 roundings of fp32 (2^-24) of scale sum |q k|, again twice."""
    b, n_q, t, d = q.shape
    n_kv = pool.bytes.shape[2]
    g = n_q // n_kv
    h = 2.0 ** -8
    out = torch.zeros((b, t, n_q, d), dtype=torch.float64)
    bound = torch.zeros_like(out)
    capacity = len(table[0]) * pool.page_rows
    for i in range(b):
        count = t if counts is None else min(max(counts[i], 0), t)
        rows = min(max(lens[i], 0), capacity)
        k, v, there = pool.dense(table[i], rows)
        for j in range(count):
            n = min(max(max(lens[i], 0) - (count - 1 - j), 0), capacity)
            seen = there[:n]
            if not bool(seen.any()):
                continue
            keys, values = k[:, :n][:, seen], v[:, :n][:, seen]
            x = q[i, :, j].double().view(n_kv, g, d)
            s = torch.matmul(x, keys.transpose(1, 2).contiguous()) * scale
            p = torch.softmax(s, -1)
            o = torch.matmul(p, values)
            off = 130 * 2.0 ** -24 * torch.matmul(x.abs(), keys.abs().transpose(1, 2).contiguous()).amax(-1, keepdim=True) * abs(scale)
            most = torch.matmul(p, values.abs())
            out[i, j] = o.view(n_q, d)
            bound[i, j] = (h * o.abs() + 2 * (h + off) * most * (1 + h) + 1e-30).view(n_q, d)
    return out, bound
