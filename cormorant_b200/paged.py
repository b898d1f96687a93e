"""The paged KV cache of a serving program: a pool of pages that sequences of
any lengths share, and the batch of rows a call works on.  ``PagedCache`` holds
the pages, ``PagedBatch`` a call's block table, row ranges and positions;
``ops.llm_paged_prep`` / ``llm_paged_attn`` / ``llm_paged_read`` take both
(corm_paged_cache in include/cormorant_b200.h).  ``PagePool`` hands pages out
on the host.

The batch's three arrays live on the device and are read there, so a captured
pass replays with what they then hold.
"""
from __future__ import annotations

import weakref
from typing import Dict, List, Optional, Sequence

import numpy as np
import torch

from . import _lib
from ._lib import CormError

PAGES = (16, 32, 64, 128, 256)     # rows of a page
WIDTHS = (16, 32, 64, 128, 256)    # head dimensions


def _bad(msg: str):
    raise CormError(_lib.CORM_EINVAL, msg)


class PagedCache:
    """``pages`` pages of ``page`` rows for KV heads of HD dimensions: kc / vc
    int8 [pages][KV][page][row bytes] and, with bits 8, ks / vs uint8
    [pages][KV][page].  ``buffers``: those tensors where the program holds them
    already; else zeros on ``device``."""

    def __init__(self, pages: int, page: int, KV: int, HD: int, bits: int = 16, device=None, buffers=None):
        if bits not in (16, 8) or page not in PAGES or HD not in WIDTHS or pages < 1 or KV < 1:
            _bad(f"PagedCache: pages {pages}, page {page} {PAGES}, KV {KV}, HD {HD} {WIDTHS}, bits {bits} (16 or 8)")
        self.pages, self.page, self.KV, self.HD, self.bits = int(pages), int(page), int(KV), int(HD), int(bits)
        rows, n = (pages, KV, page), HD * bits // 8
        if buffers is None:
            dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
            buffers = [torch.zeros(rows + (n,), dtype=torch.int8, device=dev) for _ in range(2)]
            if bits == 8:
                buffers += [torch.zeros(rows, dtype=torch.uint8, device=dev) for _ in range(2)]
        want = [(torch.int8, pages * KV * page * n)] * 2 + [(torch.uint8, pages * KV * page)] * 2
        if len(buffers) != (4 if bits == 8 else 2):
            _bad("PagedCache: kc and vc, with bits 8 also ks and vs")
        for t, (dt, numel) in zip(buffers, want):
            if t.dtype != dt or t.numel() != numel or not t.is_contiguous() or t.device != buffers[0].device:
                _bad(f"PagedCache: {numel} contiguous {dt} on one device expected, got {tuple(t.shape)} {t.dtype}")
        self.kc, self.vc = buffers[:2]
        self.ks, self.vs = buffers[2:] if bits == 8 else (None, None)
        self.device, self.index = self.kc.device, self.kc.get_device()

    def desc(self, batch: "PagedBatch") -> _lib.PagedCacheDesc:
        """The cache and the batch as the library takes them (made once for a
        pair: both keep their tensors)."""
        # (cache, descriptor), replaced as one: other threads may use the batch with theirs;
        # the cache by a weak reference: its pages are not the batch's to hold
        pair = batch._pair
        if pair is None or pair[0]() is not self:
            if batch.device != self.device:
                _bad(f"paged: the batch is on {batch.device}, the cache on {self.device}")
            ptr = [None if t is None else t.data_ptr() for t in (self.kc, self.vc, self.ks, self.vs, batch.table,
                                                                 batch.cu, batch.pos)]
            desc = _lib.PagedCacheDesc(*ptr, self.pages, self.page, self.bits, self.KV, self.HD, batch.B, batch.width,
                                       batch.rows)
            batch._pair = pair = (weakref.ref(self), desc)
        return pair[1]


class PagedBatch:
    """The packed rows of B sequences: ``table`` int32 [B][blocks] the page of
    every block, ``cu`` int32 [B + 1] the row ranges, ``pos`` int32 [B] the
    position of each sequence's first row; ``rows`` the packed rows, ``max_q``
    the most of one sequence, ``max_keys`` the most positions up to a row (a
    hint).  A batch keeps its three tensors; their contents may change between
    calls."""

    def __init__(self, table: torch.Tensor, cu: torch.Tensor, pos: torch.Tensor, rows: int, max_q: Optional[int] = None,
                 max_keys: Optional[int] = None):
        for t, nm in ((table, "table"), (cu, "cu"), (pos, "pos")):
            if t.dtype != torch.int32 or not t.is_contiguous() or t.device != table.device:
                _bad(f"PagedBatch: {nm}: contiguous int32 on one device expected, got {t.dtype} on {t.device}")
        if table.dim() != 2 or pos.numel() != table.shape[0] or cu.numel() != table.shape[0] + 1 or \
                not 0 <= rows < 1 << 31 or not 0 <= (0 if max_q is None else max_q) < 1 << 31:
            _bad(f"PagedBatch: table [B][blocks], cu [B + 1], pos [B], rows and max_q 0 .. 2^31 - 1 expected, got "
                 f"{tuple(table.shape)}, {cu.numel()}, {pos.numel()}, {rows}, {max_q}")
        self.table, self.cu, self.pos = table, cu, pos
        self.B, self.width = int(table.shape[0]), int(table.shape[1])
        self.rows = int(rows)
        self.max_q = self.rows if max_q is None else int(max_q)
        self.max_keys = 0x7FFFFFFF if max_keys is None else min(max(int(max_keys), 0), 0x7FFFFFFF)
        self.device = table.device
        self._pair = None

    @classmethod
    def of(cls, tables: Sequence[Sequence[int]], new: Sequence[int], pos: Sequence[int], device=None,
           width: Optional[int] = None) -> "PagedBatch":
        """From host lists: each sequence's pages, its new rows and the position
        of the first of them."""
        width = max([len(t) for t in tables] + [1]) if width is None else int(width)
        tab = np.full((len(tables), width), -1, np.int32)
        for b, t in enumerate(tables):
            tab[b, :len(t)] = t
        cu = np.concatenate([[0], np.cumsum(np.asarray(new, np.int64))]).astype(np.int32)
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        # one upload for the three
        flat = torch.from_numpy(np.concatenate([tab.reshape(-1), cu, np.asarray(pos, np.int32).reshape(-1)])).to(dev)
        n = tab.size
        most = max([int(p) + int(n) for p, n in zip(pos, new)] + [1])
        return cls(flat[:n].view(tab.shape), flat[n:n + cu.size], flat[n + cu.size:], rows=int(cu[-1]),
                   max_q=max([int(k) for k in new] + [0]), max_keys=most)


class PagePool:
    """Host bookkeeping of a cache's free pages: ``extend`` grows a sequence to
    a number of positions, ``release`` returns its pages."""

    def __init__(self, pages: int, page: int):
        self.page = int(page)
        self.free: List[int] = list(range(int(pages) - 1, -1, -1))
        self.held: Dict[object, List[int]] = {}

    def extend(self, seq, positions: int) -> List[int]:
        """The pages of ``seq`` covering ``positions`` rows; MemoryError, with
        nothing taken, when the pool is short."""
        have = self.held.get(seq, [])
        more = -(-int(positions) // self.page) - len(have)
        if more > len(self.free):
            raise MemoryError(f"PagePool: {more} pages wanted, {len(self.free)} free")
        have = have + [self.free.pop() for _ in range(max(more, 0))]
        self.held[seq] = have
        return have

    def release(self, seq) -> None:
        self.free.extend(reversed(self.held.pop(seq, [])))
