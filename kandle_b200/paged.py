"""A key/value cache in pages: attention over it, copies of pages, beams that share pages, and the book of free ones.

A pool holds pages of 128 positions, [pages, Hkv, 128, D]; a layer has one for keys and one for values, and one block table
[sequences, max_pages] (int32) names the page of each run of 128 positions for all of them.  The reference's only cache is contiguous
(packages/model-utils/src/kv-cache.ts:123-130); what a position holds is the same.
"""
from __future__ import annotations

import ctypes
import math
from typing import Sequence

import numpy as np

from . import core, lib
from .core import Tensor

PAGE = 128


def _r(t):
    return t._handle.ref() if t is not None else None


class Pools:
    """The pools of a model side by side, for calls that work on all of them: their descriptors are laid out once (0.7 us each)."""

    def __init__(self, tensors: Sequence[Tensor]):
        self.tensors = list(tensors)
        self.refs = lib.refs(self.tensors)

    def __len__(self) -> int:
        return len(self.tensors)


def _pools(pools) -> Pools:
    return pools if isinstance(pools, Pools) else Pools(pools)


def attention(q: Tensor, k_pool: Tensor, v_pool: Tensor, block_table: Tensor, ctx_len: Tensor, q_start: Tensor | None = None, max_query: int = 0,
              scale: float | None = None, out: Tensor | None = None) -> Tensor:
    """Attention of new tokens over a paged cache (kd_attention_paged).  q [tokens, Hq, D]: sequence b's new tokens are the rows
    q_start[b] .. q_start[b+1] (without q_start: equal shares), their keys and values already the last of its ctx_len[b] positions in the
    pages; each sees the positions up to its own.  max_query: the most new tokens of a sequence, if the program knows it.  out shares no memory with
    what is read; its rows outside the sequences stay as they are (without `out` they hold anything)."""
    if out is None:
        out = Tensor(_handle=core._output(q.shape, q.dtype))
    lib.call("kd_attention_paged", _r(q), _r(k_pool), _r(v_pool), _r(block_table), _r(ctx_len), _r(q_start), int(max_query),
             1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale), _r(out))
    return out


def copy_pages(pools, src: Tensor, dst: Tensor) -> None:
    """Page src[i] of every pool to page dst[i] (kd_kv_pages_copy)."""
    p = _pools(pools)
    lib.call("kd_kv_pages_copy", p.refs, len(p), _r(src), _r(dst))


def fork_pages(pools, parents: Tensor, block_table: Tensor, spare: Tensor, length: Tensor) -> None:
    """The beams of every request go on behind parents [requests, beams] (kd_kv_pages_fork)."""
    p = _pools(pools)
    lib.call("kd_kv_pages_fork", p.refs, len(p), _r(parents), _r(block_table), _r(spare), _r(length))


class PagePool:
    """Which pages are free, and how many sequences hold each of the others."""

    def __init__(self, pages: int):
        self.pages = int(pages)
        self.held = np.zeros(self.pages, np.int32)
        self._free = list(range(self.pages - 1, -1, -1))       # the lowest one is taken first

    @property
    def free(self) -> int:
        return len(self._free)

    def take(self, n: int) -> np.ndarray:
        if n > len(self._free):
            raise ValueError(f"Cache overflow: {n} pages are needed, {len(self._free)} of {self.pages} are free")
        got = np.array([self._free.pop() for _ in range(n)], np.int32)
        self.held[got] = 1
        return got

    def share(self, pages) -> None:
        """One more sequence holds each of these pages."""
        pages = self._known(pages)
        if (self.held[pages] == 0).any():
            raise ValueError("a free page cannot be shared")
        np.add.at(self.held, pages, 1)

    def release(self, pages) -> None:
        """One sequence fewer holds each of these pages; those that nobody holds are free again."""
        pages = self._known(pages)
        left = self.held.copy()
        np.subtract.at(left, pages, 1)
        if (left < 0).any():
            raise ValueError("a page is released that nobody holds")
        gone = np.unique(pages[left[pages] == 0])
        self.held = left
        self._free = sorted(set(self._free) | set(gone.tolist()), reverse=True)

    def keep(self, pages) -> None:
        """Exactly these pages are held from now on, by as many sequences as name each: what a program knows when the tables were changed on
        the device (fork_pages)."""
        self.held = np.bincount(self._known(pages), minlength=self.pages).astype(np.int32)
        self._free = np.flatnonzero(self.held == 0)[::-1].tolist()

    def compact(self) -> tuple[np.ndarray, np.ndarray]:
        """Moves (src, dst) after which the held pages are the first ones.  The book is that of after the moves; copy_pages makes them, and the
        tables' entries change from src to dst."""
        n = int((self.held > 0).sum())
        src, dst = np.flatnonzero(self.held[n:] > 0) + n, np.flatnonzero(self.held[:n] == 0)
        self.held[dst] = self.held[src]
        self.held[src] = 0
        self._free = list(range(self.pages - 1, n - 1, -1))
        return src.astype(np.int32), dst.astype(np.int32)

    def _known(self, pages) -> np.ndarray:
        pages = np.asarray(pages, np.int64).reshape(-1)
        if pages.size and (pages.min() < 0 or pages.max() >= self.pages):
            raise ValueError(f"pages lie between 0 and {self.pages - 1}")
        return pages
