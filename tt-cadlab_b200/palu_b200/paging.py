"""Pages of paged latent caches: reserving, forking, freeing, compacting and copying them.

A paged cache ([n_blocks, n_groups, block_size, r], ``PagedAttentionConfig``) and its page table are what the decode op
reads (``page_table``); ``PagePool`` keeps the table, the reference counts and the mapped entries on the GPU, so that
requests can be admitted, split into samples or beams, finished and defragmented without a host round trip per page. The
reference plans paged caches and has not built them (HANDOFF.md:54-55, 126-127).
"""
from __future__ import annotations

import ctypes
from array import array
from typing import Sequence

import torch

from palu_b200 import _lib

STATUS = {1: "the pool ran out of pages", 2: "a fork's parent held fewer positions than asked for",
          4: "a fork's child was not empty"}


def _ints(x, what: str) -> array:
    """Host integers as a C int array (``_at`` is its address)."""
    if isinstance(x, torch.Tensor):
        if x.is_cuda:
            raise RuntimeError(f"{what} must be on the host (a sequence or a CPU tensor)")
        x = x.reshape(-1).tolist()
    try:
        return array("i", x)
    except OverflowError:
        raise RuntimeError(f"{what} must fit 32 bits") from None


def _at(a: array) -> int:
    return a.buffer_info()[0]


def _caches(caches: Sequence[torch.Tensor]):
    """The caches as the library takes them; n_blocks."""
    if not caches:
        raise RuntimeError("at least one cache is needed")
    n_blocks, device = caches[0].shape[0], caches[0].device
    arr = (_lib.PageCache * len(caches))()
    for a, c in zip(arr, caches):
        if not c.is_cuda:
            raise RuntimeError(f"palu_b200 runs on CUDA tensors only (no CPU path); got a tensor on {c.device}")
        if c.dim() < 2 or c.shape[0] != n_blocks or c.device != device or c.numel() == 0:
            raise RuntimeError(f"caches must be [{n_blocks}, ...] tensors on {device}, got {tuple(c.shape)} on {c.device}")
        if not c[0].is_contiguous():
            raise RuntimeError("the pages of a cache must be contiguous")
        a.base, a.block_stride = c.data_ptr(), c.stride(0) * c.element_size()
        a.block_bytes = c[0].numel() * c.element_size()
    return arr, n_blocks, device


def copy_pages(caches: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]) -> None:
    """Page src[i] to page dst[i] in every cache (palu_copy_pages): ``caches`` [n_blocks, ...] tensors of any type, ``src`` /
    ``dst`` host lists. A page is copied to at most once, and not copied both from and to."""
    arr, n_blocks, device = _caches(caches)
    s, d = _ints(src, "src"), _ints(dst, "dst")
    if len(s) != len(d):
        raise RuntimeError(f"src and dst must have the same length, got {len(s)} and {len(d)}")
    with torch.cuda.device(device):
        _lib.check(_lib.load().palu_copy_pages(arr, len(arr), n_blocks, _at(s), _at(d), len(s), _lib.stream_handle(device)))


class PagePool:
    """The pages of a set of caches that share one page table (every layer's K and V): ``caches`` [n_blocks, n_groups,
    block_size, ...] tensors, ``rows`` table rows of ``blocks_per_row`` entries.

    ``table`` [rows, blocks_per_row] int32 is the page table of the decode ops (-1: no page), ``refs`` [n_blocks] how many
    entries name a page, ``mapped`` [rows] a row's entries in use; all are views of ``state``, so a copy of it is a snapshot.
    Row numbers and lengths are host integers; the pages stay on the GPU: nothing waits, and the calls can be captured
    into a CUDA graph (which then repeats them with the same rows and lengths). A page taken is always the lowest free one.
    Order the calls on one pool, and the work that reads its caches, on one stream."""

    def __init__(self, caches: Sequence[torch.Tensor], *, rows: int, blocks_per_row: int):
        caches = list(caches)
        self._caches, self.n_blocks, self.device = _caches(caches)
        sizes = {int(c.shape[2]) for c in caches if c.dim() >= 3}
        if any(c.dim() < 3 for c in caches) or len(sizes) != 1:
            raise RuntimeError("caches must be [n_blocks, n_groups, block_size, ...] tensors of one block_size")
        if rows < 1 or blocks_per_row < 1:
            raise RuntimeError(f"rows and blocks_per_row must be positive, got {rows} and {blocks_per_row}")
        self.caches, self.block_size = caches, sizes.pop()
        self.rows, self.blocks_per_row = int(rows), int(blocks_per_row)
        n = self.rows * self.blocks_per_row
        self.state = torch.zeros(n + self.n_blocks + self.rows, dtype=torch.int32, device=self.device)
        self.table = self.state[:n].view(self.rows, self.blocks_per_row)
        self.refs, self.mapped = self.state[n:n + self.n_blocks], self.state[n + self.n_blocks:]
        self.table.fill_(-1)
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        lib = _lib.load()
        self._ws = torch.empty(int(lib.palu_page_workspace_bytes(self.n_blocks)), dtype=torch.uint8, device=self.device)
        self._ws_at, self._ws_bytes, self._n_caches = self._ws.data_ptr(), self._ws.numel(), len(self._caches)
        self._pool = ctypes.byref(_lib.PagePoolInfo(self.table.data_ptr(), self.refs.data_ptr(), self.mapped.data_ptr(),
                                                    self._status.data_ptr(), self.rows, self.blocks_per_row, self.n_blocks,
                                                    self.block_size))

    def _call(self, fn, *args) -> None:
        if self.device.index != torch.cuda.current_device():
            with torch.cuda.device(self.device):
                return self._call(fn, *args)
        _lib.check(fn(self._pool, *args, _lib.stream_handle(self.device)))

    def reserve(self, rows: Sequence[int], lens: Sequence[int]) -> None:
        """Pages for positions 0 .. lens[i] - 1 of rows[i] (palu_reserve_pages); a row keeps the pages it has."""
        r, n = _ints(rows, "rows"), _ints(lens, "lens")
        if len(r) != len(n):
            raise RuntimeError(f"rows and lens must have the same length, got {len(r)} and {len(n)}")
        self._call(_lib.load().palu_reserve_pages, _at(r), _at(n), len(r))

    def fork(self, parents: Sequence[int], children: Sequence[int], lens: Sequence[int]) -> None:
        """children[i], an empty row, continues parents[i] behind its first lens[i] positions (palu_fork_pages): whole pages
        are shared (read-only from then on), a page filled only partly is copied in every cache."""
        p, c, n = _ints(parents, "parents"), _ints(children, "children"), _ints(lens, "lens")
        if not len(p) == len(c) == len(n):
            raise RuntimeError(f"parents, children and lens must have the same length, got {len(p)}, {len(c)} and {len(n)}")
        self._call(_lib.load().palu_fork_pages, self._caches, self._n_caches, _at(p), _at(c), _at(n), len(p), self._ws_at,
                   self._ws_bytes)

    def free(self, rows: Sequence[int]) -> None:
        """The rows give up their pages (palu_free_pages); a page is free once no row names it."""
        r = _ints(rows, "rows")
        self._call(_lib.load().palu_free_pages, _at(r), len(r))

    def compact(self) -> None:
        """Pages in use move to the lowest places, in every cache; table and counts follow (palu_compact_pages)."""
        self._call(_lib.load().palu_compact_pages, self._caches, self._n_caches, self._ws_at, self._ws_bytes)

    def check(self) -> None:
        """Wait, and raise RuntimeError for what went wrong in a call since the last check (pages ran out, a fork's parent
        was too short or its child not empty; such a fork was left out)."""
        st = int(self._status.item())
        if st:
            self._status.zero_()
            raise RuntimeError("page pool: " + "; ".join(t for b, t in STATUS.items() if st & b))
