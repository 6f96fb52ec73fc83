"""Residual addition and root-mean-square norm into the 8-bit activation that
a product reads (qmm_rms_norm_act): the step in front of a decoder layer's
products.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._lib import X_F32, check, lib
from .qtensor import _X_DTYPES, GgmlDType, QAct, on_device, raw_stream


class NormOut(NamedTuple):
    """What rms_norm_act gives: the quantized activation (None without a weight
    type), the stream after the addition, and the normed values (None unless asked for)."""

    act: Optional[QAct]
    h: torch.Tensor
    y: Optional[torch.Tensor]


def _rows(name: str, t: torch.Tensor, x: torch.Tensor) -> int:
    """The distance of t's rows, t checked against x."""
    if t is not x and (t.shape != x.shape or t.dtype != x.dtype or t.device != x.device):
        raise ValueError(f"rms_norm_act: {name} {tuple(t.shape)} {t.dtype} on {t.device}, x is {tuple(x.shape)} "
                         f"{x.dtype} on {x.device}")
    if t.is_contiguous():
        return t.shape[-1]
    if t.dim() != 2 or t.stride(1) != 1 or t.stride(0) < t.shape[1]:
        raise ValueError(f"rms_norm_act: {name} needs rows of consecutive values, not strides {t.stride()}")
    return t.stride(0)


def rms_norm_act(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None,
                 dtype: Optional[GgmlDType] = GgmlDType.Q4K, y_dtype: Optional[torch.dtype] = None,
                 h: Optional[torch.Tensor] = None) -> NormOut:
    """h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight, and y quantized
    for the products of `dtype` weights (None: not quantized; then y_dtype is
    needed). x and residual [..., k] in f32, f16 or bf16, their rows
    contiguous or, in two dimensions, any distance apart; weight [k] f32. h is
    rounded to x's type and the norm is that of the rounded stream. `h` names
    a tensor to write the stream to, which can be x or residual itself;
    without a residual the stream is x. y_dtype asks for y too, as f32, f16 or
    bf16. The activation equals QAct.quantize of the f32 y bit for bit."""
    code = _X_DTYPES.get(x.dtype)
    if code is None or not x.is_cuda or x.dim() < 1:
        raise ValueError(f"rms_norm_act: an f32, f16 or bf16 tensor on the GPU, not {x.dtype} on {x.device}")
    shape, device = x.shape, x.device
    k = shape[-1]
    if k < 1 or k % 4:
        raise ValueError(f"rms_norm_act: rows of {k} values (a multiple of 4 is needed)")
    if weight.dtype != torch.float32 or weight.shape != (k,) or weight.device != device or not weight.is_contiguous():
        raise ValueError(f"rms_norm_act: weight must be {k} contiguous f32 on {device}")
    if not eps >= 0.0:
        raise ValueError(f"rms_norm_act: eps {eps}")
    if dtype is None and y_dtype is None:
        raise ValueError("rms_norm_act: neither a weight type to quantize for nor y_dtype")
    if y_dtype is not None and y_dtype not in _X_DTYPES:
        raise ValueError(f"rms_norm_act: y_dtype f32, f16 or bf16, not {y_dtype}")
    xs = _rows("x", x, x)
    hp = rp = None
    rs = hs = k
    if residual is not None:
        rp, rs = residual.data_ptr(), _rows("residual", residual, x)
    if h is not None:
        hp, hs = h.data_ptr(), _rows("h", h, x)
    elif residual is not None:
        h = torch.empty(shape, dtype=x.dtype, device=device)
        hp = h.data_ptr()
    else:
        h = x
    act = QAct.alloc(shape, QAct.layout_of(dtype), device) if dtype is not None else None
    y = torch.empty(shape, dtype=y_dtype, device=device) if y_dtype is not None else None
    rows = x.numel() // k
    if rows:
        with on_device(device):
            check("qmm_rms_norm_act", lib().qmm_rms_norm_act(
                x.data_ptr(), code, xs, rp, rs, weight.data_ptr(), eps, hp, hs,
                None if act is None else act.data_.data_ptr(), 0 if act is None else act.layout,
                None if y is None else y.data_ptr(), X_F32 if y is None else _X_DTYPES[y_dtype], k, k, rows,
                raw_stream(device)))
    return NormOut(act, h, y)
