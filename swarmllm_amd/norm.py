"""Residual addition and root-mean-square norm into the 8-bit activation that
a product reads (qmm_rms_norm_act): the step in front of a decoder layer's
products (the reference's add_rmsnorm, kernels/fused_decode.cu:47-240).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._lib import X_F32, check, lib
from .qtensor import _X_DTYPES, GgmlDType, QAct, on_device


class NormOut(NamedTuple):
    """What rms_norm_act gives: the quantized activation (None without a weight
    type), the stream after the addition, and the normed values (None unless asked for)."""

    act: Optional[QAct]
    h: torch.Tensor
    y: Optional[torch.Tensor]


def _rows(name: str, t: torch.Tensor, like: torch.Tensor) -> int:
    """The distance of t's rows, checked against x (`like`)."""
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"rms_norm_act: {name} {tuple(t.shape)} {t.dtype} on {t.device}, x is {tuple(like.shape)} "
                         f"{like.dtype} on {like.device}")
    k = t.shape[-1]
    if t.is_contiguous():
        return k
    if t.dim() != 2 or t.stride(1) != 1 or t.stride(0) < k:
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
    if x.dtype not in _X_DTYPES or not x.is_cuda or x.dim() < 1:
        raise ValueError(f"rms_norm_act: an f32, f16 or bf16 tensor on the GPU, not {x.dtype} on {x.device}")
    k = x.shape[-1]
    if k < 1 or k % 4:
        raise ValueError(f"rms_norm_act: rows of {k} values (a multiple of 4 is needed)")
    if weight.dtype != torch.float32 or tuple(weight.shape) != (k,) or weight.device != x.device \
            or not weight.is_contiguous():
        raise ValueError(f"rms_norm_act: weight must be {k} contiguous f32 on {x.device}")
    if not eps >= 0.0:
        raise ValueError(f"rms_norm_act: eps {eps}")
    if dtype is None and y_dtype is None:
        raise ValueError("rms_norm_act: neither a weight type to quantize for nor y_dtype")
    if y_dtype is not None and y_dtype not in _X_DTYPES:
        raise ValueError(f"rms_norm_act: y_dtype f32, f16 or bf16, not {y_dtype}")
    xs = _rows("x", x, x)
    rs = _rows("residual", residual, x) if residual is not None else 0
    given = h
    if h is None:
        h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else x
    hs = _rows("h", h, x)
    rows = x.numel() // k
    act = QAct.alloc(x.shape, QAct.layout_of(dtype), x.device) if dtype is not None else None
    y = torch.empty(x.shape, dtype=y_dtype, device=x.device) if y_dtype is not None else None
    if rows:
        keep = residual is not None or given is not None
        with on_device(x.device):
            check("qmm_rms_norm_act", lib().qmm_rms_norm_act(
                x.data_ptr(), _X_DTYPES[x.dtype], xs, residual.data_ptr() if residual is not None else None, rs,
                weight.data_ptr(), eps, h.data_ptr() if keep else None, hs,
                act.data_.data_ptr() if act is not None else None, act.layout if act is not None else 0,
                y.data_ptr() if y is not None else None, _X_DTYPES[y_dtype] if y is not None else X_F32, k, k, rows,
                torch.cuda.current_stream().cuda_stream))
    return NormOut(act, h, y)
