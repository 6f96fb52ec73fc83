"""Tokens from logits (qmm_sample): temperature, top-k, top-p and min-p, each
request's own, from given uniform numbers.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional

import torch

from ._lib import check, lib
from .qtensor import _X_DTYPES, on_device, raw_stream


class Sampled(NamedTuple):
    """What sample gives: a token a row (int32, -1 where a row has none), and
    the chance that it was drawn with among the tokens that the settings left."""

    ids: torch.Tensor
    probs: torch.Tensor


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Optional[torch.Tensor] = None,
           top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
           min_p: Optional[torch.Tensor] = None) -> Sampled:
    """A token for each row of logits [rows, vocab] (f32, f16 or bf16, rows any
    distance apart) from a uniform number u [rows] in [0, 1). temperature, top_p
    and min_p [rows] f32 and top_k [rows] int32, None for off: weights
    exp((x - max x) / temperature) (0: the largest logit's token); of the tokens
    the top_k largest stay, of those the fewest that hold top_p of their
    weight, of those the ones of at least min_p of the largest weight. The token
    is the first, by index, at which the running sum of the weights left passes u
    of their total; equal logits count by index, the lowest first. -inf and NaN
    are never drawn; a row of nothing else gives -1 and 0. The ids viewed as
    uint32 are what QTensor.gather_rows takes. A row's token does not depend on
    the other rows."""
    code, device = _X_DTYPES.get(logits.dtype), logits.device
    if code is None or logits.dim() != 2 or not logits.is_cuda:
        raise ValueError(f"sample: logits [rows, vocab] f32, f16 or bf16 on the GPU, not {logits.dtype} "
                         f"{tuple(logits.shape)} on {device}")
    rows, vocab = logits.shape
    if not 1 <= vocab <= 1 << 19 or rows > 65535:
        raise ValueError(f"sample: {rows} rows of {vocab} logits (at most 65535 of 1 to 2^19)")
    stride = logits.stride(0) if rows > 1 else vocab
    if (vocab > 1 and logits.stride(1) != 1) or stride < vocab:
        raise ValueError(f"sample: logits need rows of consecutive values, not strides {logits.stride()}")
    ptrs = []
    for name, t, dtype in (("u", u, torch.float32), ("temperature", temperature, torch.float32),
                           ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                           ("min_p", min_p, torch.float32)):
        if t is None and name != "u":
            ptrs.append(None)
            continue
        if t is None or t.dtype != dtype or t.shape != (rows,) or t.device != device or not t.is_contiguous():
            raise ValueError(f"sample: {name} must be {rows} contiguous {dtype} on {device}")
        ptrs.append(t.data_ptr())
    ids = torch.empty(rows, dtype=torch.int32, device=device)
    probs = torch.empty(rows, dtype=torch.float32, device=device)
    if rows:
        with on_device(device):
            need = _need(device.index, vocab, rows, top_k is not None or top_p is not None or min_p is not None)
            size = ctypes.c_size_t(need)
            # a buffer a call: stream-ordered, and under capture the graph's own
            ws = torch.empty(need, dtype=torch.uint8, device=device)
            check("qmm_sample", lib().qmm_sample(logits.data_ptr(), code, stride, *ptrs, ids.data_ptr(), probs.data_ptr(),
                                                 vocab, rows, ws.data_ptr(), need, ctypes.byref(size), 1,
                                                 raw_stream(device)))
    return Sampled(ids, probs)


@functools.lru_cache(maxsize=1024)
def _need(device: int, vocab: int, rows: int, settings: bool) -> int:
    """The workspace bytes that qmm_sample plans on the current device (`device`): by the sizes, and whether a setting
    but the temperature is given."""
    need, some = ctypes.c_size_t(0), 256 if settings else None  # any address: planning reads none
    check("qmm_sample", lib().qmm_sample(None, 0, vocab, None, None, some, None, None, None, None, vocab, rows, None, 0,
                                         ctypes.byref(need), 0, 0))
    return need.value
