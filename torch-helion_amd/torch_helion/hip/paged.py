"""A paged key/value cache for sequences of their own lengths, and the decode step over it.

The reference has no KV cache (its models/llama_block.py:82-105 recomputes every key). Here
``PagedKVCache`` holds the pages of all layers and the page table that the paged entry points
of ``ops`` read; which page belongs to whom is decided on the host by ``PageBook``. Sequences
that were forked share pages until one of them writes into a shared one, which it copies
first. ``PagedDecodeBlock`` is the decode step of ``DecodeBlock`` for a batch whose rows stand
at positions of their own:

  k0  th_gemm e4m3        [q | k | v] = r (x g1) [Wq | Wk | Wv], in fp32
  k1  th_paged_append     q = rope(q);  the cache's pages = rope(k), v
  k2  th_paged_attention  over keys 0 .. position of each row
  k3 .. k5                as k2 .. k4 of DecodeBlock

Positions and page table are device tensors, so one captured graph serves every step.
"""

from __future__ import annotations

import heapq
import math
from typing import Iterable

import torch

from . import abi, ops
from .decode import DecodeBlock


def _refuse(entry: str, message: str) -> None:
    raise abi.HipBackendError(entry, abi.TH_ERR_INVALID, message)


class PageBook:
    """Which sequence (row) holds which pages, and how many rows hold each page. Every change is
    whole or not at all: a call that would run out of pages or rows raises and changes nothing."""

    def __init__(self, pages: int, page_size: int, rows: int, row_pages: int) -> None:
        self.page_size, self.row_pages = page_size, row_pages
        self.refs = [0] * pages
        self.free = list(range(pages))                 # a heap: the lowest page is taken first
        self.free_rows = list(range(rows))
        self.pages: dict[int, list[int]] = {}          # open row -> its pages in order
        self.length: dict[int, int] = {}               # open row -> its tokens

    def _check(self, row: int, entry: str) -> None:
        if row not in self.pages:
            _refuse(entry, f"row {row} is not open")

    def open(self) -> int:
        if not self.free_rows:
            _refuse("PagedKVCache.open", "no free row")
        row = heapq.heappop(self.free_rows)
        self.pages[row], self.length[row] = [], 0
        return row

    def fork(self, row: int) -> int:
        self._check(row, "PagedKVCache.fork")
        new = self.open()
        self.pages[new], self.length[new] = list(self.pages[row]), self.length[row]
        for page in self.pages[new]:
            self.refs[page] += 1
        return new

    def _drop(self, page: int) -> None:
        self.refs[page] -= 1
        if self.refs[page] == 0:
            heapq.heappush(self.free, page)

    def close(self, row: int) -> None:
        self._check(row, "PagedKVCache.close")
        for page in self.pages.pop(row):
            self._drop(page)
        del self.length[row]
        heapq.heappush(self.free_rows, row)

    def extend(self, counts: dict[int, int]) -> tuple[list[tuple[int, int]], list[tuple[int, int, int]]]:
        """Room for ``counts[row]`` more tokens of each row. Returns the page copies (from, to) that
        rows need which would write into a shared page, and the page table's new entries (row,
        index, page)."""
        entry, size = "PagedKVCache.extend", self.page_size
        grow, shared = [], {}                          # (row, pages to add); rows whose last page is shared
        sharers: dict[int, int] = {}
        for row, n in counts.items():
            self._check(row, entry)
            if n < 0:
                _refuse(entry, f"row {row}: {n} tokens")
            need = -(-(self.length[row] + n) // size)
            if need > self.row_pages:
                _refuse(entry, f"row {row}: {self.length[row] + n} tokens exceed the table's {self.row_pages * size}")
            grow.append((row, need - len(self.pages[row])))
            at = self.length[row] // size
            if n and self.length[row] % size:
                page = self.pages[row][at]
                # the last of a page's holders to come writes in place
                if self.refs[page] - sharers.get(page, 0) > 1:
                    sharers[page] = sharers.get(page, 0) + 1
                    shared[row] = at
        if sum(n for _, n in grow) + len(shared) > len(self.free):
            _refuse(entry, f"{sum(n for _, n in grow) + len(shared)} pages needed, {len(self.free)} free")
        copies, entries = [], []
        for row, at in shared.items():
            old, new = self.pages[row][at], heapq.heappop(self.free)
            self.refs[new] = 1
            self.refs[old] -= 1
            self.pages[row][at] = new
            copies.append((old, new))
            entries.append((row, at, new))
        for row, n in grow:
            for _ in range(n):
                page = heapq.heappop(self.free)
                self.refs[page] = 1
                entries.append((row, len(self.pages[row]), page))
                self.pages[row].append(page)
            self.length[row] += counts[row]
        return copies, entries

    def shrink(self, row: int, length: int) -> None:
        """Drop the tokens of a row past ``length`` and the pages that held only them."""
        self._check(row, "PagedKVCache.shrink")
        if not 0 <= length <= self.length[row]:
            _refuse("PagedKVCache.shrink", f"row {row} has {self.length[row]} tokens, not {length}")
        keep = -(-length // self.page_size)
        for page in self.pages[row][keep:]:
            self._drop(page)
        del self.pages[row][keep:]
        self.length[row] = length

    def compact(self) -> list[tuple[int, int]]:
        """Move the pages in use down to pages 0 .. used - 1: the moves (from, to), each onto a free
        page, the highest pages in use into the lowest free ones."""
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if self.refs[p] == 0]
        movers = [p for p in range(used, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[a], self.refs[b] = 0, self.refs[a]
        for row in self.pages.values():
            row[:] = [to.get(p, p) for p in row]
        self.free = list(range(used, len(self.refs)))
        return list(to.items())


class PagedKVCache:
    """The pages ``k``, ``v`` [layers, pages, page_size, kv_heads, head_dim] of all layers and the
    int32 page table [rows, ceil(max_len / page_size)] on the device, -1 past each row's pages.

    ``dtype`` is torch.bfloat16 or torch.float8_e4m3fn; an e4m3 cache may have scales, fp32
    [layers, kv_heads]. ``page_size`` is a power of two of at least 16; ``attend`` takes a
    ``head_dim`` of 64 or 128, the other calls any up to 1024. Calls work on the current stream;
    ``extend``, ``fork``, ``shrink``, ``close`` and ``compact`` change the table there, so calls that
    read it must be ordered with them, as calls on one stream are. An ``extend`` that needs pages and
    a ``compact`` that moves some copy their page numbers from the host and wait for the stream."""

    def __init__(self, *, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, rows: int, max_len: int,
                 dtype: torch.dtype = torch.bfloat16, device: int | torch.device = 0, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None) -> None:
        entry = "PagedKVCache"
        self.device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if self.device.type != "cuda":
            _refuse(entry, f"device {device} is not a HIP device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        if min(layers, pages, kv_heads, head_dim, rows, max_len) <= 0:
            _refuse(entry, "sizes must be positive")
        if page_size < 16 or page_size & (page_size - 1):
            _refuse(entry, f"page_size {page_size} must be a power of two of at least 16")
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            _refuse(entry, f"no cache of {dtype}")
        for s in (k_scale, v_scale):
            if s is not None and (dtype != torch.float8_e4m3fn or s.shape != (layers, kv_heads) or s.dtype != torch.float32):
                _refuse(entry, "scales are fp32 [layers, kv_heads] of an e4m3 cache")
        shape = (layers, pages, page_size, kv_heads, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=self.device)
        self.v = torch.zeros_like(self.k)
        self.k_scale = None if k_scale is None else k_scale.to(self.device).contiguous()
        self.v_scale = None if v_scale is None else v_scale.to(self.device).contiguous()
        self.page_table = torch.full((rows, -(-max_len // page_size)), -1, dtype=torch.int32, device=self.device)
        self.book = PageBook(pages, page_size, rows, self.page_table.shape[1])

    # ------------------------------------------------------------------ sequences
    @property
    def free_pages(self) -> int:
        return len(self.book.free)

    def length(self, row: int) -> int:
        self.book._check(row, "PagedKVCache.length")
        return self.book.length[row]

    def open(self) -> int:
        """A row for a new, empty sequence."""
        return self.book.open()

    def close(self, row: int) -> None:
        """Give the row back, and its pages that no other row holds."""
        self.book.close(row)
        self.page_table[row].fill_(-1)

    def extend(self, counts: dict[int, int] | Iterable[int]) -> None:
        """Room for ``counts[row]`` more tokens of each row (for one each of the rows of a list),
        which the caller then appends at the positions that follow. A row that shares the page it
        will write into gets a copy of it. Raises, and changes nothing, without enough pages."""
        if not isinstance(counts, dict):
            rows = list(counts)
            counts = dict.fromkeys(rows, 1)
            if len(counts) != len(rows):
                _refuse("PagedKVCache.extend", "a row is listed twice")
        copies, entries = self.book.extend(counts)
        if copies:
            self._copy(copies)
        self._write(entries)

    def shrink(self, row: int, length: int) -> None:
        """Drop the row's tokens past ``length`` (a rejected speculation, a trimmed prompt)."""
        self.book.shrink(row, length)
        self.page_table[row, len(self.book.pages[row]):].fill_(-1)

    def fork(self, row: int) -> int:
        """A new row with the same tokens, which shares its pages."""
        new = self.book.fork(row)
        self.page_table[new] = self.page_table[row]
        return new

    def compact(self) -> int:
        """Move the pages in use to the front of the pool; returns how many they are (the pages
        behind them are free). One launch moves them in every layer and renames the table."""
        moves = self.book.compact()
        if moves:
            page_map = torch.arange(len(self.book.refs), dtype=torch.int32)
            for a, b in moves:
                page_map[a] = b
            self._copy(moves, page_map.to(self.device))
        return len(self.book.refs) - len(self.book.free)

    def _copy(self, pairs: list[tuple[int, int]], page_map: torch.Tensor | None = None) -> None:
        src, dst = torch.tensor(pairs, dtype=torch.int32).t().contiguous().to(self.device)
        ops.copy_pages(self.k, self.v, src, dst, page_table=None if page_map is None else self.page_table, page_map=page_map)

    def _write(self, entries: list[tuple[int, int, int]]) -> None:
        if entries:
            row, at, page = torch.tensor(entries, dtype=torch.int64).t().contiguous().to(self.device)
            self.page_table[row, at] = page.to(torch.int32)

    # ------------------------------------------------------------------ one layer's calls
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, **options) -> None:
        """``ops.paged_append`` on a layer's pages (its ``rows``, ``freqs``, ``q``, ... as options)."""
        ops.paged_append(k, v, positions, self.k[layer], self.v[layer], self.page_table, **self._scales(layer), **options)

    def attend(self, layer: int, q: torch.Tensor, positions: torch.Tensor, out: torch.Tensor, *, max_keys: int | None = None,
               **options) -> torch.Tensor:
        """``ops.paged_attention`` on a layer's pages (its ``scale``, ``rows``, ``window``, ... as options).
        ``max_keys``: a bound on the keys that any of the tokens sees, such as the longest row's length;
        later pages are not looked at, and short rows take a faster form."""
        table = self.page_table
        if max_keys is not None:
            if max_keys <= 0:
                _refuse("PagedKVCache.attend", f"max_keys {max_keys} must be positive")
            table = table[:, :-(-max_keys // self.k.shape[2])]
        return ops.paged_attention(q, self.k[layer], self.v[layer], table, positions, out, **self._scales(layer), **options)

    def _scales(self, layer: int) -> dict[str, torch.Tensor]:
        return {n: s[layer] for n, s in (("k_scale", self.k_scale), ("v_scale", self.v_scale)) if s is not None}


class PagedDecodeBlock(DecodeBlock):
    """The decode step of a Llama block over one layer of a ``PagedKVCache``: row i of the batch
    stands at ``positions[i]`` of the cache's row ``rows[i]`` (row i without ``rows``); a negative
    position marks an unused row of the batch, for which nothing is stored and whose output is
    the block's for an attention of zeros.

    ``freqs`` (``ops.rope_frequencies``; by default those of ``rope_theta``) and ``rope_scale`` give
    the rotary positions, ``window`` and ``softcap`` the attention's."""

    def __init__(self, state_dict: dict[str, torch.Tensor], *, hidden: int, heads: int, kv_heads: int, intermediate: int,
                 eps: float, rope_theta: float, batch: int, cache: PagedKVCache, layer: int = 0,
                 freqs: torch.Tensor | None = None, rope_scale: float = 1.0, window: int = 0, softcap: float = 0.0,
                 fold_gain: bool = True) -> None:
        if (cache.k.shape[3], cache.k.shape[4]) != (kv_heads, hidden // heads) or not 0 <= layer < cache.k.shape[0]:
            _refuse("PagedDecodeBlock", f"layer {layer} of a cache {tuple(cache.k.shape)} does not fit {kv_heads} heads of "
                                        f"{hidden // heads}")
        self.cache, self.layer = cache, layer
        self.rope_scale, self.window, self.softcap = rope_scale, window, softcap
        self.freqs = ops.rope_frequencies(hidden // heads, rope_theta) if freqs is None else freqs
        max_len = cache.page_table.shape[1] * cache.k.shape[2]
        with torch.cuda.device(cache.device):
            super().__init__(state_dict, hidden=hidden, heads=heads, kv_heads=kv_heads, intermediate=intermediate, eps=eps,
                             rope_theta=rope_theta, batch=batch, max_len=max_len, device=cache.device, fold_gain=fold_gain)

    def _allocate_cache(self) -> None:
        self.freqs = self.freqs.to(self.device)
        self.qkv = torch.empty(self.B, (self.H + 2 * self.Hkv) * self.hd, device=self.device)
        n = ops.paged_attention_workspace_bytes(self.B, self.H, self.Hkv, self.hd, self.max_len, window=self.window,
                                                dtype=self.cache.k.dtype, device=self.device)
        self.attn_ws = torch.empty(n, dtype=torch.uint8, device=self.device)
        self.n_invalid = torch.zeros(1, dtype=torch.int32, device=self.device)   # tokens that no page had room for

    def step(self, x: torch.Tensor, positions: torch.Tensor, rows: torch.Tensor | None = None) -> torch.Tensor:
        """One token per row; x [batch, hidden] bf16, positions (and rows) int32 [batch], all on the
        device. The cache must have room at the positions (``PagedKVCache.extend``; a token
        without is not stored and counted in ``self.n_invalid``). Returns the block output [batch, hidden] (bf16; ``self.out32`` holds it in fp32)."""
        if x.dtype != torch.bfloat16 or tuple(x.shape) != (self.B, self.D):
            _refuse("PagedDecodeBlock.step", "x must be bf16 [batch, hidden]")
        if torch.cuda.current_device() != self.device.index:   # th_gemm launches on the current device
            with torch.cuda.device(self.device):
                return self.step(x, positions, rows)
        self._gemm(self.wqkv, x, [ops.EpiSpec(abi.EPI_ACC, self.qkv, a=0)], rscale_mask=0b1, lhs_gain=self.g1, sumsq=True,
                   inv_k=1.0 / self.D, eps=self.eps)
        qw, kvw = self.H * self.hd, self.Hkv * self.hd
        q, k, v = self.qkv.split([qw, kvw, kvw], 1)
        self.cache.append(self.layer, k, v, positions, rows=rows, freqs=self.freqs, rope_scale=self.rope_scale, q=q,
                          q_out=self.q, n_invalid=self.n_invalid)
        self.cache.attend(self.layer, self.q, positions, self.attn, rows=rows, scale=1.0 / math.sqrt(self.hd),
                          window=self.window, softcap=self.softcap, workspace=self.attn_ws)
        return self._after_attention(x)

    def capture(self, x: torch.Tensor, positions: torch.Tensor, rows: torch.Tensor | None = None) -> None:
        """Record ``step`` into a HIP graph; ``replay()`` then runs it on whatever x, positions, rows
        and the cache's page table hold by then. The recording itself stores nothing: it is made
        with every position at -1, and ``positions`` has its values back afterwards."""
        with torch.cuda.device(self.device):
            held = positions.clone()
            positions.fill_(-1)
            try:
                torch.cuda.synchronize()
                self.step(x, positions, rows)
                torch.cuda.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    self.step(x, positions, rows)
            finally:
                positions.copy_(held)
            torch.cuda.synchronize()
        self.graph = g

    def bytes_per_step(self, positions: Iterable[int]) -> int:
        """HBM bytes a step at these positions must move: every weight byte and the keys and values
        that each row sees."""
        seen = (min(p + 1, self.window) if self.window else p + 1 for p in positions)
        row = 2 * self.Hkv * self.hd * self.cache.k.element_size()
        return self.weight_bytes() + sum(max(n, 0) for n in seen) * row
