"""Low-rank adapters of many requests beside a shared projection
(qmm_adapters_add): each row of a batch with its own request's adapter.
"""
from __future__ import annotations

import ctypes
import functools
from typing import List, Optional, Sequence, Tuple

import torch

from ._lib import QMM_OK, QMM_UNSUPPORTED, Adapter, check, lib
from .qtensor import _X_DTYPES, on_device, raw_stream

_MOST = 4  # projections a call


class Adapters:
    """The adapters of one projection [n, k]: a [slots, rank, k] and b [slots, n,
    rank] of one type (f32, f16 or bf16), scales [slots] f32 (None: 1). rank is a
    multiple of 8 up to 128; an adapter of a lower rank has zeros behind it. k is a
    multiple of 32, slots at most 4096."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scales: Optional[torch.Tensor] = None):
        if a.dim() != 3 or b.dim() != 3 or a.dtype not in _X_DTYPES or a.shape[0] != b.shape[0] \
                or a.shape[1] != b.shape[2]:
            raise ValueError(f"Adapters: a [slots, rank, k] and b [slots, n, rank] f32, f16 or bf16, not {a.dtype} "
                             f"{tuple(a.shape)} and {b.dtype} {tuple(b.shape)}")
        self.slots, self.rank, self.k = a.shape
        self.n = b.shape[1]
        self.device, self.dtype = a.device, a.dtype
        for name, t in (("a", a), ("b", b)):
            if t.dtype != a.dtype or not t.is_contiguous() or not t.is_cuda or t.device != self.device \
                    or t.data_ptr() % 16:
                raise ValueError(f"Adapters: {name} must be contiguous, 16-byte aligned {a.dtype} on one GPU, not "
                                 f"{t.dtype} {tuple(t.shape)} on {t.device}")
        if self.rank < 8 or self.rank > 128 or self.rank % 8 or self.k < 32 or self.k % 32 or self.n < 1 \
                or self.slots > 4096:
            raise ValueError(f"Adapters: {self.slots} of rank {self.rank} (at most 4096, a multiple of 8 up to 128) for a "
                             f"projection [{self.n}, {self.k}] (k a multiple of 32)")
        if scales is not None and (scales.dtype != torch.float32 or scales.shape != (self.slots,)
                                   or scales.device != self.device or not scales.is_contiguous()):
            raise ValueError(f"Adapters: scales must be {self.slots} contiguous f32 on {self.device}")
        self.a, self.b, self.scales = a, b, scales
        self._ptrs = (a.data_ptr(), b.data_ptr(), None if scales is None else scales.data_ptr())

    def add(self, y: torch.Tensor, x: torch.Tensor, ids: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """out = y + scales[i] * (x a[i]^T) b[i]^T row by row, i = ids[row]; a row
        whose id is outside [0, slots) is y's. y [..., n] f32 is the projection's
        product of x [..., k] (f32, f16 or bf16), ids int32 one a row; out: by
        default y itself, which is added to; otherwise it shares no memory with
        what the call reads (other columns of one wide array share none). The
        products are of x's and the adapters' own values, with f32 sums."""
        return Adapters.add_shared([y], x, [self], ids, None if out is None else [out])[0]

    @staticmethod
    def add_shared(ys: Sequence[torch.Tensor], x: torch.Tensor, adapters: Sequence["Adapters"], ids: torch.Tensor,
                   outs: Optional[Sequence[torch.Tensor]] = None) -> List[torch.Tensor]:
        """Adapters.add for up to four projections of one x (q, k and v; gate and
        up): the counterpart of QMatMul.forward_shared. The adapters have one
        number of slots and one type."""
        outs = list(ys) if outs is None else list(outs)
        count = len(adapters)
        if not 1 <= count <= _MOST or len(ys) != count or len(outs) != count:
            raise ValueError(f"Adapters.add_shared: 1 to {_MOST} projections, not {count} with {len(ys)} y and {len(outs)} out")
        first = adapters[0]
        device, k, x_type = first.device, first.k, _X_DTYPES.get(x.dtype)
        if x_type is None or x.device != device or x.dim() < 1 or x.shape[-1] != k:
            raise ValueError(f"Adapters.add: x [..., {k}] f32, f16 or bf16 on {device}, not {x.dtype} {tuple(x.shape)} on "
                             f"{x.device}")
        rows = x.numel() // k
        if ids.dtype != torch.int32 or ids.numel() != rows or ids.device != device or not ids.is_contiguous():
            raise ValueError(f"Adapters.add: ids must be {rows} contiguous int32 on {device}, not {ids.dtype} "
                             f"{tuple(ids.shape)} on {ids.device}")
        xs = _rows("x", x, k)
        c = (Adapter * count)()
        for i, (ad, y, out) in enumerate(zip(adapters, ys, outs)):
            if ad.device != device or ad.dtype != first.dtype or ad.slots != first.slots or ad.k != k:
                raise ValueError(f"Adapters.add_shared: {ad!r} beside {first!r}")
            for name, t in (("y", y), ("out", out)):
                if t.dtype != torch.float32 or t.device != device or t.shape != (*x.shape[:-1], ad.n):
                    raise ValueError(f"Adapters.add: {name} {[*x.shape[:-1], ad.n]} f32 on {device}, not {t.dtype} "
                                     f"{tuple(t.shape)} on {t.device}")
            c[i] = Adapter(*ad._ptrs, y.data_ptr(), out.data_ptr(), ad.n, _rows("y", y, ad.n), _rows("out", out, ad.n),
                           ad.rank)
        if rows == 0:
            return outs
        with on_device(device):
            need = _need(device.index, first.slots, k, rows, tuple((ad.n, ad.rank) for ad in adapters))
            size = ctypes.c_size_t(need)
            # a buffer a call: stream-ordered, and under capture the graph's own
            ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
            status = lib().qmm_adapters_add(
                count, c, first.slots, _X_DTYPES[first.dtype], x.data_ptr(), x_type, xs, ids.data_ptr(), k, rows,
                None if ws is None else ws.data_ptr(), need, ctypes.byref(size), 1, raw_stream(device))
        if status == QMM_UNSUPPORTED:  # (the arrays' places are the library's to check: a call is host time)
            raise ValueError("Adapters.add: an out that shares memory with x, ids, an adapter, another projection's y or "
                             "out, or with its own y without being it")
        if status != QMM_OK:
            check("qmm_adapters_add", status)
        return outs

    def __repr__(self) -> str:
        return f"Adapters[{self.slots} of rank {self.rank} for [{self.n}, {self.k}]; {self.dtype}]"


def _rows(name: str, t: torch.Tensor, width: int) -> int:
    """The distance of t's rows."""
    if t.is_contiguous():
        return width
    if t.dim() != 2 or (width > 1 and t.stride(1) != 1) or t.stride(0) < width:
        raise ValueError(f"Adapters.add: {name} needs rows of consecutive values, not strides {t.stride()}")
    return t.stride(0)


@functools.lru_cache(maxsize=1024)
def _need(device: int, slots: int, k: int, rows: int, sizes: Tuple[Tuple[int, int], ...]) -> int:
    """The workspace bytes that qmm_adapters_add plans on the current device (`device`): by the sizes alone."""
    c, need = (Adapter * len(sizes))(), ctypes.c_size_t(0)
    for i, (n, rank) in enumerate(sizes):
        c[i] = Adapter(None, None, None, None, None, n, n, n, rank)
    check("qmm_adapters_add", lib().qmm_adapters_add(len(sizes), c, slots, _X_DTYPES[torch.float32], None,
                                                     _X_DTYPES[torch.float32], k, None, k, rows, None, 0,
                                                     ctypes.byref(need), 0, 0))
    return need.value
