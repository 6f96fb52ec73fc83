"""A paged key/value cache in Q8_0 and the attention over it (qmm_cache_* and
qmm_attend): what stands between a decoder layer's q/k/v and o products.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple

import torch

from ._lib import X_F16, Cache, QmmError, check, lib
from .qtensor import _X_DTYPES, on_device, raw_stream


class KvCache:
    """Pages of `page` positions for kv_heads heads of head_dim values, keys
    and values quantized per 32 values of a head (an f16 scale, 8-bit codes):

      k_codes int8 [pages, kv_heads, page, head_dim], k_scales f16 [.., page, head_dim / 32]
      v_codes int8 [pages, kv_heads, head_dim, page], v_scales f16 [.., head_dim / 32, page]

    Position p of a sequence lies in slot table[p // page] * page + p % page
    of its page table. Which pages a sequence has is the caller's to keep."""

    def __init__(self, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor):
        if k_codes.dim() != 4:
            raise ValueError(f"KvCache: k_codes [pages, kv_heads, page, head_dim], not {tuple(k_codes.shape)}")
        pages, heads, page, hd = k_codes.shape
        self.device = k_codes.device
        ptrs = []
        for name, t, shape, dt in (("k_codes", k_codes, (pages, heads, page, hd), torch.int8),
                                   ("k_scales", k_scales, (pages, heads, page, hd // 32), torch.float16),
                                   ("v_codes", v_codes, (pages, heads, hd, page), torch.int8),
                                   ("v_scales", v_scales, (pages, heads, hd // 32, page), torch.float16)):
            ptrs.append(t.data_ptr())
            if t.dtype != dt or t.shape != shape or not t.is_contiguous() or not t.is_cuda \
                    or t.device != self.device or ptrs[-1] % 16:
                raise ValueError(f"KvCache: {name} must be contiguous, 16-byte aligned {dt} {shape} on one GPU, not "
                                 f"{t.dtype} {tuple(t.shape)} on {t.device}")
        _plane_bytes(pages, heads, hd, page)
        self.planes = (k_codes, k_scales, v_codes, v_scales)
        self.pages, self.kv_heads, self.page, self.head_dim = pages, heads, page, hd
        self._c = Cache(*ptrs, pages, heads, hd, page)
        self._ref = ctypes.byref(self._c)

    @staticmethod
    def alloc(pages: int, kv_heads: int, head_dim: int, page: int = 64, device="cuda") -> "KvCache":
        """A cache of zeros: head_dim 64, 96, 128 or 256, page 16 to 256 (a power of two)."""
        _plane_bytes(pages, kv_heads, head_dim, page)
        return KvCache(torch.zeros((pages, kv_heads, page, head_dim), dtype=torch.int8, device=device),
                       torch.zeros((pages, kv_heads, page, head_dim // 32), dtype=torch.float16, device=device),
                       torch.zeros((pages, kv_heads, head_dim, page), dtype=torch.int8, device=device),
                       torch.zeros((pages, kv_heads, head_dim // 32, page), dtype=torch.float16, device=device))

    def slots(self, table: torch.Tensor, start: int, count: int) -> torch.Tensor:
        """The slots (int64) of positions start .. start + count - 1 of the sequence with this page table (1-D),
        all of them inside it. A page id outside the cache gives slots outside it."""
        if table.dim() != 1 or start < 0 or count < 0 or start + count > table.numel() * self.page:
            raise ValueError(f"KvCache.slots: positions {start} .. {start + count - 1} of a table {tuple(table.shape)} of "
                             f"pages of {self.page}")
        p = torch.arange(start, start + count, device=table.device)
        return table.long()[p // self.page] * self.page + p % self.page

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantizes keys and values [tokens, kv_heads, head_dim] (f32, f16 or
        bf16; the last axis contiguous, the others any distance apart) into
        `slots` (int64 [tokens]). A negative slot, or one past the cache,
        writes nothing; the others are distinct."""
        tokens = slots.numel()
        self._slots("write", slots)
        shape, code = (tokens, self.kv_heads, self.head_dim), _X_DTYPES.get(k.dtype)
        if code is None or k.shape != shape or v.shape != shape or v.dtype != k.dtype or k.device != self.device \
                or v.device != self.device:
            raise ValueError(f"KvCache.write: k and v {list(shape)} in f32, f16 or bf16 on {self.device}, not {k.dtype} "
                             f"{tuple(k.shape)} on {k.device} and {v.dtype} {tuple(v.shape)} on {v.device}")
        if tokens == 0:
            return
        ks, khs = self._strides("write", "k", k)
        vs, vhs = self._strides("write", "v", v)
        with on_device(self.device):
            check("qmm_cache_write", lib().qmm_cache_write(self._ref, k.data_ptr(), ks, khs, v.data_ptr(), vs, vhs,
                                                           code, slots.data_ptr(), tokens,
                                                           raw_stream(self.device)))

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
        """The keys and values [tokens, kv_heads, head_dim] of `slots` (int64
        [tokens]) as f16, bf16 or f32; zeros for a slot outside the cache."""
        self._slots("read", slots)
        if dtype not in _X_DTYPES:
            raise ValueError(f"KvCache.read: f32, f16 or bf16, not {dtype}")
        tokens = slots.numel()
        k = torch.empty((tokens, self.kv_heads, self.head_dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        if tokens:
            with on_device(self.device):
                check("qmm_cache_read", lib().qmm_cache_read(self._ref, slots.data_ptr(), tokens, k.data_ptr(),
                                                             v.data_ptr(), _X_DTYPES[dtype],
                                                             raw_stream(self.device)))
        return k, v

    def attend(self, q: torch.Tensor, q_starts: torch.Tensor, kv_lens: torch.Tensor, tables: torch.Tensor,
               max_q: int, max_kv: Optional[int] = None, scale: Optional[float] = None, window: int = 0,
               sinks: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """Causal attention of the new tokens q [tokens, heads, head_dim] (f16,
        bf16 or f32) over the cached positions of their sequences, the new ones
        among them (write them first). Sequence b's new tokens are rows
        q_starts[b] .. q_starts[b + 1] - 1, the last of its kv_lens[b] cached
        positions; tables [seqs, pages a sequence] names its pages (all int32).
        max_q and max_kv: at least the most new tokens and cached positions of
        a sequence (max_kv: by default what a row of tables holds); they choose
        the launch and cut what is longer. scale: by default head_dim ** -0.5.
        window > 0: a token sees the last `window` positions, its own among
        them. sinks [heads] f32: a term exp(sink) in each softmax's sum. Rows
        of q that belong to no sequence are left as they were in `out` (as
        torch.empty gives them without one). The products run on f16 operands
        with f32 sums: an f32 q is rounded to f16, as is a bf16 one (f32 outputs
        end about 5.5e-4 from exact ones). A row does
        not depend on the other sequences' values; its last bits can follow from
        max_q, max_kv, the number of sequences and, past 256 query rows a kv
        head, the other sequences' lengths, by which the sums are split."""
        device = self.device
        q_type = _X_DTYPES.get(q.dtype)
        if q.dim() != 3 or q_type is None or q.device != device or q.shape[2] != self.head_dim or q.shape[1] < 1 \
                or q.shape[1] % self.kv_heads:
            raise ValueError(f"KvCache.attend: q [tokens, a multiple of {self.kv_heads} heads, {self.head_dim}] f16, "
                             f"bf16 or f32 on {device}, not {q.dtype} {tuple(q.shape)} on {q.device}")
        tokens, heads, hd = q.shape
        seqs = kv_lens.numel()
        self._int32("q_starts", q_starts, (seqs + 1,))
        self._int32("kv_lens", kv_lens, (seqs,))
        if tables.dim() != 2:
            raise ValueError(f"KvCache.attend: tables [{seqs}, pages a sequence], not {tuple(tables.shape)}")
        pages = tables.shape[1]
        self._int32("tables", tables, (seqs, pages))
        if max_q < 0 or window < 0 or (max_kv is not None and max_kv < 0):
            raise ValueError(f"KvCache.attend: max_q {max_q}, max_kv {max_kv}, window {window}")
        if sinks is not None and (sinks.dtype != torch.float32 or sinks.shape != (heads,) or sinks.device != device
                                  or not sinks.is_contiguous()):
            raise ValueError(f"KvCache.attend: sinks must be {heads} contiguous f32 on {device}")
        out_stride = heads * hd
        if out is None:
            out_type = q_type if out_dtype is None else _X_DTYPES.get(out_dtype)
            if out_type is None:
                raise ValueError(f"KvCache.attend: out_dtype f16, bf16 or f32, not {out_dtype}")
            out = torch.empty((tokens, heads, hd), dtype=out_dtype or q.dtype, device=device)
        else:
            out_type = _X_DTYPES.get(out.dtype)
            if out_type is None or (out_dtype is not None and out.dtype != out_dtype) or out.device != device \
                    or out.shape != (tokens, heads, hd) \
                    or (tokens and (out.stride(2) != 1 or (heads > 1 and out.stride(1) != hd))) \
                    or (tokens > 1 and out.stride(0) < out_stride):
                raise ValueError(f"KvCache.attend: out [{tokens}, {heads}, {hd}] {out_dtype or 'f16, bf16 or f32'}, "
                                 f"rows of consecutive values, not {out.dtype} {tuple(out.shape)} strides "
                                 f"{out.stride()}")
            if tokens > 1:
                out_stride = out.stride(0)
        if tokens == 0 or seqs == 0:
            return out
        qs, qhs = self._strides("attend", "q", q)
        if max_kv is None:
            max_kv = pages * self.page
        with on_device(device):
            need = _attend_need(device.index, self.pages, self.kv_heads, hd, self.page, tokens, heads, pages, seqs,
                                max_q, max_kv, window)
            size = ctypes.c_size_t(need)
            # a buffer a call: stream-ordered, and under capture the graph's own
            ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
            check("qmm_attend", lib().qmm_attend(
                self._ref, q.data_ptr(), q_type, qs, qhs, tokens, heads, q_starts.data_ptr(), kv_lens.data_ptr(),
                tables.data_ptr(), pages, seqs, max_q, max_kv, hd ** -0.5 if scale is None else scale, window,
                None if sinks is None else sinks.data_ptr(), out.data_ptr(), out_type, out_stride,
                None if ws is None else ws.data_ptr(), need, ctypes.byref(size), 1, raw_stream(device)))
        return out

    def _int32(self, name: str, t: torch.Tensor, shape) -> None:
        if t.dtype != torch.int32 or t.shape != shape or t.device != self.device or not t.is_contiguous():
            raise ValueError(f"KvCache.attend: {name} must be contiguous int32 {shape} on {self.device}, not {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")

    def _slots(self, name: str, slots: torch.Tensor) -> None:
        if slots.dtype != torch.int64 or slots.dim() != 1 or slots.device != self.device or not slots.is_contiguous():
            raise ValueError(f"KvCache.{name}: slots must be contiguous int64 [tokens] on {self.device}, not "
                             f"{slots.dtype} {tuple(slots.shape)} on {slots.device}")

    def _strides(self, name: str, what: str, t: torch.Tensor) -> Tuple[int, int]:
        """Distances of the tokens and heads of t [tokens, heads, head_dim]."""
        ts, hs, ds = t.stride()
        if t.shape[0] <= 1:
            ts = t.shape[1] * self.head_dim
        if t.shape[1] <= 1:
            hs = self.head_dim
        if ds != 1 or hs < self.head_dim or ts < 0:
            raise ValueError(f"KvCache.{name}: {what} needs heads of {self.head_dim} consecutive values, not strides "
                             f"{t.stride()}")
        return ts, hs

    def __repr__(self) -> str:
        return f"KvCache[{self.pages} pages of {self.page}, {self.kv_heads} heads of {self.head_dim}; Q8_0]"


@functools.lru_cache(maxsize=1024)
def _attend_need(device: int, pages: int, kv_heads: int, head_dim: int, page: int, tokens: int, heads: int,
                 table_pages: int, seqs: int, max_q: int, max_kv: int, window: int) -> int:
    """The workspace bytes that qmm_attend plans on the current device (`device`): by the sizes alone."""
    some = 256  # any aligned address: planning reads none
    c, need = Cache(some, some, some, some, pages, kv_heads, head_dim, page), ctypes.c_size_t(0)
    row = heads * head_dim
    check("qmm_attend", lib().qmm_attend(ctypes.byref(c), None, X_F16, row, head_dim, tokens, heads, None, None, None,
                                         table_pages, seqs, max_q, max_kv, 1.0, window, None, None, X_F16, row, None,
                                         0, ctypes.byref(need), 0, 0))
    return need.value


@functools.lru_cache(maxsize=64)
def _plane_bytes(pages: int, kv_heads: int, head_dim: int, page: int) -> Tuple[int, int]:
    """Bytes of a codes and of a scales plane; ValueError for sizes not covered."""
    codes, scales = ctypes.c_size_t(0), ctypes.c_size_t(0)
    try:
        check("qmm_cache_plane_bytes", lib().qmm_cache_plane_bytes(pages, kv_heads, head_dim, page,
                                                                   ctypes.byref(codes), ctypes.byref(scales)))
    except QmmError:
        raise ValueError(f"KvCache: {pages} pages of {page} for {kv_heads} heads of {head_dim}: pages of 16 to 256 "
                         "positions (a power of two), heads of 64, 96, 128 or 256 values") from None
    return codes.value, scales.value
