"""The page tables of a batch's sequences, kept on the device, and the rows that
a step of the batch has (qmm_pages_step): what a serving loop does between two
forward passes, without the host knowing a length.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from ._lib import Pages, check, lib
from .qtensor import on_device, raw_stream


class BatchRows(NamedTuple):
    """What PageTables.step gives: where each sequence's rows begin (KvCache.attend's
    q_starts), the tokens that each sequence took, and of every row its cache
    slot (KvCache.write's), its position and its sequence."""

    q_starts: torch.Tensor
    taken: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    seq: torch.Tensor


class PageTables:
    """The page tables [seqs, pages a sequence] and lengths [seqs] of a batch's
    sequences, and a stack of the pages that none of them holds (all int32):
    `free` [pool], of which the first free_count [1] entries count. KvCache.attend
    takes `tables` and `lens` as they are; a page is one sequence's, the same in
    every layer's cache."""

    def __init__(self, tables: torch.Tensor, lens: torch.Tensor, free: torch.Tensor, free_count: torch.Tensor, page: int):
        if tables.dim() != 2:
            raise ValueError(f"PageTables: tables [seqs, pages a sequence], not {tuple(tables.shape)}")
        seqs, row = tables.shape
        self.device = tables.device
        for name, t, shape in (("tables", tables, (seqs, row)), ("lens", lens, (seqs,)), ("free", free, (free.numel(),)),
                               ("free_count", free_count, (1,))):
            if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous() or not t.is_cuda \
                    or t.device != self.device:
                raise ValueError(f"PageTables: {name} must be contiguous int32 {shape} on one GPU, not {t.dtype} "
                                 f"{tuple(t.shape)} on {t.device}")
        if page < 16 or page > 256 or page & (page - 1) or seqs > 4096 or row * page > 1 << 30 or seqs * row > 1 << 30 \
                or free.numel() >= 1 << 31:
            raise ValueError(f"PageTables: {seqs} sequences of {row} pages of {page}: at most 4096, pages of 16 to 256 "
                             "positions (a power of two), 2^30 positions a sequence, 2^30 entries, fewer than 2^31 pages")
        self.tables, self.lens, self.free, self.free_count = tables, lens, free, free_count
        self.seqs, self.row_pages, self.page = seqs, row, page
        self._c = Pages(tables.data_ptr(), lens.data_ptr(), free.data_ptr(), free_count.data_ptr(), row, row, free.numel(),
                        seqs, page)
        self._ref = ctypes.byref(self._c)

    @staticmethod
    def alloc(seqs: int, row_pages: int, pool: int, page: int = 64, device="cuda") -> "PageTables":
        """Empty sequences of up to row_pages pages each, and `pool` free pages (0 .. pool - 1, the first taken first)."""
        return PageTables(torch.full((seqs, row_pages), -1, dtype=torch.int32, device=device),
                          torch.zeros(seqs, dtype=torch.int32, device=device),
                          torch.arange(pool - 1, -1, -1, dtype=torch.int32, device=device),
                          torch.full((1,), pool, dtype=torch.int32, device=device), page)

    def step(self, new: Optional[torch.Tensor] = None, tokens: int = 0, keep: Optional[torch.Tensor] = None) -> BatchRows:
        """Each sequence is cut to its first keep[b] positions (None: not cut; a
        keep below 0 or past its length cuts nothing), the pages behind them
        freed (0: it is finished, or its place a new one's), and then given pages
        for new[b] more tokens (None: none). keep and new: int32 [seqs]. The
        batch has `tokens` rows, the sequences' one after another; rows past
        them have slot, position and sequence -1. A sequence whose rows, row of
        the table or pages do not suffice is not extended (taken 0, its rows'
        slots and positions -1), and once pages have run out no sequence behind
        it takes one. Updates tables, lens, free and free_count in place."""
        for name, t in (("new", new), ("keep", keep)):
            if t is not None and (t.dtype != torch.int32 or t.shape != (self.seqs,) or t.device != self.device
                                  or not t.is_contiguous()):
                raise ValueError(f"PageTables.step: {name} must be contiguous int32 [{self.seqs}] on {self.device}, not "
                                 f"{t.dtype} {tuple(t.shape)} on {t.device}")
        if tokens < 0 or tokens > 1 << 29:
            raise ValueError(f"PageTables.step: {tokens} tokens")
        device = self.device
        slots = torch.empty(tokens, dtype=torch.int64, device=device)
        # (two allocations for the five: a call is host time)
        q_starts, taken, positions, seq = torch.empty(2 * (self.seqs + tokens) + 1, dtype=torch.int32, device=device) \
            .split_with_sizes([self.seqs + 1, self.seqs, tokens, tokens])
        with on_device(device):
            check("qmm_pages_step", lib().qmm_pages_step(
                self._ref, None if keep is None else keep.data_ptr(), None if new is None else new.data_ptr(), tokens,
                q_starts.data_ptr(), taken.data_ptr(), slots.data_ptr(), positions.data_ptr(), seq.data_ptr(),
                raw_stream(device)))
        return BatchRows(q_starts, taken, slots, positions, seq)

    def __repr__(self) -> str:
        return f"PageTables[{self.seqs} sequences of {self.row_pages} pages of {self.page}; {self.free.numel()} pages]"
