"""Pages of the KV cache: which sequence holds which, sharing them between forks,
and copying them on the device.

``KVPagePool`` keeps the books on the host (a reference count per page, a table
per sequence) and moves data with ``ie_copy_pages``: one launch copies a list of
pages in every layer's K and V.  A fork shares the parent's whole pages and gets
its own copy of the last, partly filled one, so every page that a sequence may
still write belongs to it alone.  Pages are given out lowest number first, so
the same calls always give the same tables.

The copies run on the current stream (or ``stream=``); a caller that reads or
writes the cache on another stream orders the two itself.
"""
from __future__ import annotations

import ctypes
import heapq

import numpy as np

from . import _lib
from .device import require_cuda


class OutOfPages(RuntimeError):
    """The pool has fewer free pages than the call needs; nothing was changed."""


def _page_numbers(name: str, pages) -> np.ndarray:
    """A list or array of page numbers as int32; what int32 cannot hold as it is (floats,
    numbers beyond its range) is refused, not cast."""
    a = np.asarray(pages)
    if a.dtype == np.int32:          # the library checks the range
        return np.ascontiguousarray(a)
    if a.size == 0:
        return np.zeros(a.shape, dtype=np.int32)
    if a.dtype.kind not in "iu":
        raise ValueError(f"{name} must hold integers, not {a.dtype}")
    low, high = int(a.min()), int(a.max())
    if low < 0 or high > 0x7FFFFFFF:
        raise ValueError(f"{name} holds page {low if low < 0 else high}")
    return np.ascontiguousarray(a, dtype=np.int32)


class _Sequence:
    __slots__ = ("pages", "length")

    def __init__(self, pages: list[int], length: int):
        self.pages = pages        # page of every block, -1 where it was given back
        self.length = length      # tokens


class KVPagePool:
    def __init__(self, k_caches, v_caches, block_size: int):
        torch = require_cuda()
        caches = [*k_caches, *v_caches]
        if len(k_caches) != len(v_caches) or not caches:
            raise ValueError("one K and one V cache per layer")
        first = caches[0]
        if block_size < 1 or first.dim() != 3 or first.shape[0] % block_size:
            raise ValueError("caches are [num_blocks * block_size, kv_heads, head_dim]")
        for c in caches:
            if c.shape != first.shape or c.dtype != first.dtype or c.device != first.device \
                    or not c.is_contiguous() or not c.is_cuda:
                raise ValueError("the caches must be contiguous CUDA tensors of one shape, dtype "
                                 "and device")
        self.block_size = block_size
        self.num_pages = first.shape[0] // block_size
        self.page_bytes = block_size * first[0].numel() * first.element_size()
        self.device = first.device
        self._caches = caches     # alive as long as their addresses are used
        self._pointers = (ctypes.c_void_p * len(caches))(*[c.data_ptr() for c in caches])
        self._torch = torch
        self._refs = np.zeros(self.num_pages, dtype=np.int32)
        self._free = list(range(self.num_pages))
        self._sequences: dict[int, _Sequence] = {}
        self._next = 0

    # ---- device ---------------------------------------------------------------
    def copy_pages(self, src, dst, stream=None) -> None:
        """Page ``dst[i]`` becomes a copy of page ``src[i]`` in every cache.  A page
        written twice, or both read and written, or a number that is no page of the
        cache, is a ``ValueError``.  (The sequences' tables do not change.)"""
        src, dst = _page_numbers("src", src), _page_numbers("dst", dst)
        if src.ndim != 1 or src.shape != dst.shape:
            raise ValueError("src and dst must be lists of one length")
        if src.size == 0:
            return
        cuda = self._torch.cuda
        if self.device.index != cuda.current_device():
            with cuda.device(self.device):
                return self.copy_pages(src, dst, stream)
        _lib.check(_lib.lib().ie_copy_pages(
            self._pointers, len(self._caches), self.page_bytes, self.num_pages,
            src.ctypes.data, dst.ctypes.data, src.size, _lib.stream_ptr(stream)), "copy_pages")

    # ---- books ------------------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _sequence(self, seq: int) -> _Sequence:
        if seq not in self._sequences:
            raise ValueError(f"no sequence {seq} in this pool")
        return self._sequences[seq]

    def _take(self, count: int) -> list[int]:
        if count > len(self._free):
            raise OutOfPages(f"{count} pages wanted, {len(self._free)} free")
        pages = [heapq.heappop(self._free) for _ in range(count)]
        self._refs[pages] = 1
        return pages

    def _release(self, pages) -> None:
        for page in pages:
            if page < 0:
                continue
            self._refs[page] -= 1
            if self._refs[page] == 0:
                heapq.heappush(self._free, page)

    def new(self, tokens: int = 0) -> int:
        """A new sequence with room for ``tokens`` tokens; its number."""
        if tokens < 0:
            raise ValueError(f"a sequence of {tokens} tokens")
        pages = self._take(-(-tokens // self.block_size))
        self._sequences[self._next] = _Sequence(pages, tokens)
        self._next += 1
        return self._next - 1

    def append(self, seq: int, tokens: int = 1) -> None:
        """Room for ``tokens`` more tokens."""
        if tokens < 0:
            raise ValueError(f"cannot append {tokens} tokens")
        s = self._sequence(seq)
        s.pages += self._take(-(-(s.length + tokens) // self.block_size) - len(s.pages))
        s.length += tokens

    def fork(self, seq: int, count: int = 1, stream=None) -> list[int]:
        """``count`` sequences that continue ``seq``: its whole pages are shared, its
        last, partly filled page is copied for each (one launch)."""
        if count < 0:
            raise ValueError(f"cannot fork {count} times")
        s = self._sequence(seq)
        whole = s.length // self.block_size
        tail = [p for p in s.pages[whole:] if p >= 0]     # at most one
        own = self._take(count * len(tail))
        try:
            if own:
                self.copy_pages(tail * count, own, stream)
        except Exception:
            self._release(own)
            raise
        shared = s.pages[:whole]
        live = [p for p in shared if p >= 0]
        self._refs[live] += count
        children = []
        for i in range(count):
            mine = [own[i]] if tail else [-1] * (len(s.pages) - whole)
            self._sequences[self._next] = _Sequence(shared + mine, s.length)
            children.append(self._next)
            self._next += 1
        return children

    def free(self, seqs) -> None:
        """Gives the sequences' pages back (those that no other sequence shares)."""
        seqs = list(seqs) if hasattr(seqs, "__iter__") else [seqs]
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is freed once")
        for s in [self._sequence(n) for n in seqs]:
            self._release(s.pages)
        for n in seqs:
            del self._sequences[n]

    def trim(self, seq: int, window: int, sinks: int = 0) -> int:
        """Gives back the pages that no query from the next token on can see under
        ``window_attention(window=, sinks=)``; their entries read -1.  Returns
        how many entries were cleared."""
        if window < 1 or sinks < 0:
            raise ValueError("trim needs a window of at least 1 and sinks of at least 0")
        s = self._sequence(seq)
        # the next token is at position s.length and sees keys above s.length - window
        first = -(-sinks // self.block_size)
        last = max(0, s.length - window + 1) // self.block_size
        gone = [b for b in range(first, min(last, len(s.pages))) if s.pages[b] >= 0]
        self._release([s.pages[b] for b in gone])
        for b in gone:
            s.pages[b] = -1
        return len(gone)

    def compact(self, stream=None) -> int:
        """Moves the pages in use to the lowest numbers (one launch) and rewrites every
        table, so that the pool's upper pages are free; returns how many moved.
        Tables handed out before are stale afterwards."""
        live = np.flatnonzero(self._refs)
        src = live[live >= live.size]
        dst = np.flatnonzero(self._refs[:live.size] == 0)
        if src.size:
            self.copy_pages(src, dst, stream)
            self._refs[dst] = self._refs[src]
            self._refs[src] = 0
            moved = dict(zip(src.tolist(), dst.tolist()))
            for s in self._sequences.values():
                s.pages = [moved.get(p, p) for p in s.pages]
            self._free = list(range(live.size, self.num_pages))
        return int(src.size)

    # ---- what attention and the cache writes take ---------------------------------
    def length(self, seq: int) -> int:
        return self._sequence(seq).length

    def pages(self, seq: int) -> list[int]:
        return list(self._sequence(seq).pages)

    def tables(self, seqs):
        """int32 [sequences, blocks] block tables on the device, padded with -1."""
        rows = [self._sequence(n).pages for n in seqs]
        out = np.full((len(rows), max([1, *map(len, rows)])), -1, dtype=np.int32)
        for i, row in enumerate(rows):
            out[i, :len(row)] = row
        return self._torch.from_numpy(out).to(self.device)

    def slot(self, seq: int, position: int) -> int:
        """Cache slot of a position of the sequence."""
        s = self._sequence(seq)
        if not 0 <= position < s.length or s.pages[position // self.block_size] < 0:
            raise ValueError(f"position {position} of sequence {seq} has no page")
        return s.pages[position // self.block_size] * self.block_size + position % self.block_size
