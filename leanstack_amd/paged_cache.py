"""Keys and values of many requests in 8 bits, in pages that requests share.

One resident pool holds pages of ``page_rows`` rows for every layer and kv head
(include/leanstack_amd.h has the format: 16 rows of a head are a block of e4m3 bytes
with one exponent): 2 x 128 bytes and an eighth per row, head and layer, half of
what ``ArenaKVCache`` takes, and only for rows that are there.  The kernels see
the pool, a page table and lengths on the device; which request has which page is
kept here, on the host:

    cache = PagedKVCache(36, 8, num_pages=4096, device="cuda")
    a = cache.open()
    cache.reserve([a], 300)                  # pages for 300 more rows
    table, lens = cache.batch([a], new=300)  # what the kernels read
    kernels.paged_append(cache, layer, k, v, table, lens)       # every layer
    kernels.paged_attention(q, cache, layer, table, lens, scale)
    cache.advance([a], 300)
    b = cache.fork(a)                        # shares a's pages
    cache.close(a)

Pages have a count of the requests that hold them.  A page that several hold is
copied before one of them writes into it (``reserve``).  ``truncate`` drops rows of
rejected drafts, ``compact`` moves the pages in use to the pool's front.  One thread at
a time keeps a cache's accounts; page tables and lengths that were made are tensors of their own.
"""

from __future__ import annotations

import torch

BLOCK_ROWS = 16
BLOCK_BYTES = 16 * 128
HEAD_DIM = 128
MAX_PAGE_ROWS = 1024


class Request:
    """One request's pages, in the order of its rows, and how many rows are written."""

    __slots__ = ("pages", "rows")

    def __init__(self) -> None:
        self.pages: list[int] = []
        self.rows = 0


class PagedKVCache:
    """The pool and the requests' pages.

    storage: uint8 [L, 2, pages, n_kv, page_rows / 16, 2048] (keys, then values, of each
    layer); exponents: uint8 [L, 2, pages, n_kv, page_rows / 16]."""

    def __init__(self, num_layers: int, num_key_value_heads: int, num_pages: int, *, page_rows: int = 64,
                 device: torch.device | str = "cpu") -> None:
        if min(num_layers, num_key_value_heads, num_pages) < 1:
            raise ValueError(f"layers, kv heads and pages must all be >= 1, got "
                             f"{(num_layers, num_key_value_heads, num_pages)}")
        if page_rows < BLOCK_ROWS or page_rows > MAX_PAGE_ROWS or page_rows & (page_rows - 1):
            raise ValueError(f"page_rows must be a power of two, {BLOCK_ROWS}..{MAX_PAGE_ROWS}, got {page_rows}")
        shape = (num_layers, 2, num_pages, num_key_value_heads, page_rows // BLOCK_ROWS)
        self._own(torch.zeros((*shape, BLOCK_BYTES), dtype=torch.uint8, device=device),
                  torch.zeros(shape, dtype=torch.uint8, device=device))

    @classmethod
    def of(cls, storage: torch.Tensor, exponents: torch.Tensor) -> "PagedKVCache":
        """The cache over an existing pool, worked in place; all its pages are free."""
        blocks = storage.shape[4] if storage.dim() == 6 else 0
        if storage.dtype is not torch.uint8 or exponents.dtype is not torch.uint8 or storage.dim() != 6 \
                or storage.shape[5] != BLOCK_BYTES or storage.shape[1] != 2 or storage.numel() == 0 \
                or exponents.shape != storage.shape[:5] or blocks & (blocks - 1) or blocks * BLOCK_ROWS > MAX_PAGE_ROWS:
            raise ValueError(f"a pool is uint8 [L, 2, pages, n_kv, 1, 2, 4 .. {MAX_PAGE_ROWS // BLOCK_ROWS}, {BLOCK_BYTES}] "
                             f"bytes and the same of exponents without the last axis, got {storage.dtype} "
                             f"{tuple(storage.shape)} and {exponents.dtype} {tuple(exponents.shape)}")
        if not (storage.is_contiguous() and exponents.is_contiguous()) or storage.device != exponents.device:
            raise ValueError("storage and exponents must be contiguous, on one device")
        cache = cls.__new__(cls)
        cache._own(storage, exponents)
        return cache

    def _own(self, storage: torch.Tensor, exponents: torch.Tensor) -> None:
        self.storage, self.exponents = storage, exponents
        self.num_layers, _, self.num_pages, self.num_key_value_heads, page_blocks, _ = storage.shape
        self.page_rows = page_blocks * BLOCK_ROWS
        self._holders = [0] * self.num_pages
        self._free = list(range(self.num_pages - 1, -1, -1))  # the lowest is taken first
        self._requests: dict[Request, None] = {}  # the open ones, in their order

    # -- pages ------------------------------------------------------------------

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def holders(self, page: int) -> int:
        """How many open requests hold a page."""
        return self._holders[page]

    def _known(self, requests: list[Request]) -> None:
        for r in requests:
            if not isinstance(r, Request) or r not in self._requests:
                raise ValueError("the request is not open in this cache")

    def open(self) -> Request:
        """A request without rows."""
        r = Request()
        self._requests[r] = None
        return r

    def close(self, request: Request) -> None:
        """The request ends: pages that no other holds are free."""
        self._known([request])
        self._release(request.pages)
        request.pages, request.rows = [], 0
        del self._requests[request]

    def _release(self, pages: list[int]) -> None:
        freed = False
        for page in pages:
            self._holders[page] -= 1
            if self._holders[page] == 0:
                self._free.append(page)
                freed = True
        if freed:
            self._free.sort(reverse=True)

    def fork(self, request: Request) -> Request:
        """A request with the same rows.  Its pages are the same until one of the two
        writes into the last, which reserve() copies."""
        self._known([request])
        other = self.open()
        other.pages = request.pages[: -(-request.rows // self.page_rows)]
        other.rows = request.rows
        for page in other.pages:
            self._holders[page] += 1
        return other

    def truncate(self, request: Request, rows: int) -> None:
        """Drop the request's rows from `rows` on, and pages without rows."""
        self._known([request])
        if not 0 <= rows <= request.rows:
            raise ValueError(f"cannot cut a request of {request.rows} rows to {rows}")
        keep = -(-rows // self.page_rows)
        self._release(request.pages[keep:])
        request.pages, request.rows = request.pages[:keep], rows

    def reserve(self, requests: list[Request], new: int | list[int]) -> None:
        """Pages for `new` more rows of each request, and none of the pages that these
        rows go to held by another (a begun one is copied, all layers, on the current
        stream).  Nothing changes if the free pages do not suffice."""
        counts = self._counts(requests, new)
        wanted, begun = [], []
        for r, n in zip(requests, counts):
            last = r.rows // self.page_rows
            shared = n > 0 and r.rows % self.page_rows != 0 and self._holders[r.pages[last]] > 1
            begun.append(shared)
            wanted.append(max(0, -(-(r.rows + n) // self.page_rows) - len(r.pages)))
        # (of several requests that share a begun page, the last to be served keeps it)
        holders: dict[int, int] = {}
        copies = []
        for r, shared in zip(requests, begun):
            if shared:
                page = r.pages[r.rows // self.page_rows]
                left = holders.setdefault(page, self._holders[page])
                if left > 1:
                    holders[page] = left - 1
                    copies.append(r)
        if sum(wanted) + len(copies) > len(self._free):
            raise ValueError(f"{sum(wanted) + len(copies)} pages are needed, {len(self._free)} are free")
        src, dst = [], []
        for r in copies:
            at = r.rows // self.page_rows
            old, page = r.pages[at], self._take()
            src.append(old)
            dst.append(page)
            r.pages[at] = page
            self._holders[old] -= 1
        for r, n in zip(requests, wanted):
            r.pages.extend(self._take() for _ in range(n))
        self._copy(src, dst)

    def _take(self) -> int:
        page = self._free.pop()
        self._holders[page] = 1
        return page

    def _counts(self, requests: list[Request], new: int | list[int]) -> list[int]:
        self._known(requests)
        if len({id(r) for r in requests}) != len(requests):
            raise ValueError("a request is named twice")
        counts = [new] * len(requests) if isinstance(new, int) else list(new)
        if len(counts) != len(requests) or any(n < 0 for n in counts):
            raise ValueError(f"one number of new rows (>= 0) per request is needed, got {counts}")
        return counts

    def _reserved(self, requests: list[Request], counts: list[int]) -> None:
        for r, n in zip(requests, counts):
            if r.rows + n > len(r.pages) * self.page_rows:
                raise ValueError(f"{r.rows} + {n} rows do not fit the request's {len(r.pages)} pages: reserve them first")

    def _copy(self, src: list[int], dst: list[int]) -> None:
        if not src:
            return
        if self.storage.is_cuda:
            from . import kernels
            moved = torch.tensor([src, dst], dtype=torch.int32, device=self.storage.device)
            kernels.copy_pages(self, moved[0], moved[1])
        else:  # (a pool in host memory: the accounting without a GPU)
            self.storage[:, :, dst] = self.storage[:, :, src]
            self.exponents[:, :, dst] = self.exponents[:, :, src]

    def advance(self, requests: list[Request], new: int | list[int]) -> None:
        """Count rows that were appended (in every layer)."""
        counts = self._counts(requests, new)
        self._reserved(requests, counts)
        for r, n in zip(requests, counts):
            r.rows += n

    def compact(self) -> int:
        """Move the pages in use to the pool's front (all layers, on the current stream);
        returns how many they are.  Page tables made before are void."""
        used = self.num_pages - len(self._free)
        holes = sorted(page for page in self._free if page < used)
        moved = [page for page in range(used, self.num_pages) if self._holders[page]]
        names = dict(zip(moved, holes))
        self._copy(moved, holes)
        for old, page in names.items():
            self._holders[page], self._holders[old] = self._holders[old], 0
        for r in self._requests:
            r.pages = [names.get(page, page) for page in r.pages]
        self._free = list(range(self.num_pages - 1, used - 1, -1))
        return used

    # -- what the kernels read ----------------------------------------------------

    def batch(self, requests: list[Request], new: int | list[int] = 0, *, table: torch.Tensor | None = None,
              lens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """(table int32 [B, pages], lens int32 [B]) of the requests on the pool's device:
        their pages, -1 behind the last, and their rows with `new` ones that a step appends.
        table / lens: existing tensors to fill (a captured step's), wide enough."""
        counts = self._counts(requests, new)
        self._reserved(requests, counts)
        for r, n in zip(requests, counts):  # (a fork since reserve(); only the begun page can be another's too)
            if n > 0 and r.rows % self.page_rows and self._holders[r.pages[r.rows // self.page_rows]] > 1:
                raise ValueError(f"row {r.rows} would go to a page that another request holds: reserve it first")
        width = max([1] + [len(r.pages) for r in requests])
        if table is not None:
            if table.dim() != 2 or table.shape[0] != len(requests) or table.shape[1] < width or table.dtype is not torch.int32:
                raise ValueError(f"table must be int32 [{len(requests)}, {width} or more], got {table.dtype} "
                                 f"{tuple(table.shape)}")
            width = table.shape[1]
        if lens is not None and (lens.shape != (len(requests),) or lens.dtype is not torch.int32):
            raise ValueError(f"lens must be int32 [{len(requests)}], got {lens.dtype} {tuple(lens.shape)}")
        rows = torch.tensor([r.pages + [-1] * (width - len(r.pages)) for r in requests], dtype=torch.int32)
        rows = rows.view(len(requests), width)
        counted = torch.tensor([r.rows + n for r, n in zip(requests, counts)], dtype=torch.int32)
        device = self.storage.device
        table = rows.to(device) if table is None else table.copy_(rows)
        lens = counted.to(device) if lens is None else lens.copy_(counted)
        return table, lens

    def export(self, request: Request, cache) -> None:
        """The request's rows appended to an ArenaKVCache (exact: stored values are bf16
        numbers), for a request that goes on alone in a captured decode step.  Nothing is
        written if they do not fit."""
        from . import kernels
        self._known([request])
        layers, _, heads, capacity, dim = cache.storage.shape
        if (layers, heads, dim) != (self.num_layers, self.num_key_value_heads, HEAD_DIM):
            raise ValueError(f"a cache of {self.num_layers} layers and {self.num_key_value_heads} kv heads of {HEAD_DIM} is "
                             f"needed, got {layers} layers and {heads} heads of {dim}")
        for layer, rows in enumerate(cache.layer_seq_lens):
            if rows + request.rows > capacity:
                raise ValueError(f"layer {layer}: {rows} + {request.rows} rows have no room in {capacity}")
        if not request.rows:
            return
        table, lens = self.batch([request])
        starts = torch.zeros_like(lens)
        for layer in range(self.num_layers):
            keys, values = kernels.paged_read(self, layer, table, starts, request.rows, lens=lens)
            cache.write_rows(layer, keys, values)
