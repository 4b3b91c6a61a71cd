"""Products with 4-bit weights and group scales (batch-1 decode and small batches).

    qweight, scales, zeros = quantize_w4(weight)          # once, when a model is loaded
    y = w4_linear(x, qweight, scales, zeros)              # every token

A weight is scale * (code - zero): codes 0..15, two to a byte (the even input in the low half), a
scale and optionally a zero point for every group of 32, 64 or 128 consecutive inputs of an output.
The compute is the hand-written gfx950 kernel behind `mq_w4_linear` (include/megaqwen_hip.h,
megaqwen_amd/csrc/w4.hip); there is no PyTorch fallback.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._launch import DTYPES, call, no_grad

GROUP_SIZES = (32, 64, 128)
_HALF = (torch.float16, torch.bfloat16)


def quantize_w4(weight: torch.Tensor, group_size: int = 128, *, symmetric: bool = True,
                scale_dtype: torch.dtype = torch.bfloat16
                ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(qweight uint8 [N, K/2], scales [N, K/group_size], zeros uint8 [N, K/group_size] or None) of
    a weight [N, K], by rounding to the nearest code; for load time, on any device.

    symmetric: scale = max|w| / 7 of a group and codes 8 + round(w / scale).  Otherwise the range of
    a group (with 0) is spread over the 16 codes: scale = (max - min) / 15, zero = round(-min /
    scale).  A group of zeros has scale 0."""
    if weight.ndim != 2 or not weight.is_floating_point():
        raise ValueError(f"expected a floating-point weight [N, K], got {weight.dtype} {tuple(weight.shape)}")
    if group_size not in GROUP_SIZES or weight.shape[1] % group_size != 0 or weight.shape[1] == 0:
        raise ValueError(f"group_size must be one of {GROUP_SIZES} and divide K = {weight.shape[1]}, "
                         f"got {group_size}")
    if scale_dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"scale_dtype must be bfloat16 or float16, got {scale_dtype}")
    w = weight.detach().float().unflatten(1, (-1, group_size))
    if symmetric:
        scale = (w.abs().amax(-1) / 7.0).to(scale_dtype)
        zero = None
    else:
        low, high = w.amin(-1).clamp_max(0.0), w.amax(-1).clamp_min(0.0)
        scale = ((high - low) / 15.0).to(scale_dtype)
        zero = torch.where(scale > 0, -low / scale.float(), 0.0).round().clamp(0, 15)
    s = scale.float().unsqueeze(-1)
    q = torch.where(s > 0, w / s, 0.0).round() + (8.0 if zero is None else zero.unsqueeze(-1))
    u = q.clamp(0, 15).to(torch.uint8).flatten(1)
    return (u[:, 0::2] | (u[:, 1::2] << 4)).contiguous(), scale, None if zero is None else zero.to(torch.uint8)


def w4_linear(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor,
              zeros: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
              out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x W^T (+ residual) for x [..., K] (bf16 or fp16) and a 4-bit weight [N, K].

    qweight: uint8 [N, K/2]; scales: bf16 or fp16 [N, K/group] (the group size, 32, 64 or 128,
    follows from the shapes); zeros: uint8 [N, K/group], 8 everywhere if None.  The result has x's
    type, or fp32 with out_dtype=torch.float32 (logits); `residual` [..., N] of that type is added
    before its one rounding.  Sums are fp32.  Meant for up to about 64 rows of x (one pass over the
    weights per 64 rows); more rows are computed all the same."""
    # (the checks are most of a short product's call: plain comparisons, the message in _refuse)
    dtype, dev = x.dtype, x.get_device()
    if not x.is_cuda or dtype not in _HALF or qweight.ndim != 2 or qweight.dtype != torch.uint8 \
            or scales.ndim != 2 or scales.dtype not in _HALF:
        _refuse(x, qweight, scales, zeros, residual, out_dtype)
    (n, half), (sn, groups), shape = qweight.shape, scales.shape, x.shape
    k = 2 * half
    if not shape or shape[-1] != k or sn != n or groups < 1 or k % groups != 0 or k // groups not in GROUP_SIZES \
            or qweight.get_device() != dev or scales.get_device() != dev \
            or not (qweight.is_contiguous() and scales.is_contiguous()):
        _refuse(x, qweight, scales, zeros, residual, out_dtype)
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape
                              or zeros.get_device() != dev or not zeros.is_contiguous()):
        _refuse(x, qweight, scales, zeros, residual, out_dtype)
    if out_dtype is None:
        out_dtype = dtype
    elif out_dtype != dtype and out_dtype != torch.float32:
        _refuse(x, qweight, scales, zeros, residual, out_dtype)
    size = (shape[0], n) if len(shape) == 2 else (*shape[:-1], n)
    if residual is not None and (residual.dtype != out_dtype or residual.shape != size or residual.get_device() != dev):
        _refuse(x, qweight, scales, zeros, residual, out_dtype)
    if torch.is_grad_enabled():
        no_grad("w4_linear", x, scales, residual)
    out = x.new_empty(size) if out_dtype == dtype else x.new_empty(size, dtype=out_dtype)
    if out.numel() == 0:
        return out
    x = x.contiguous()
    at = x.data_ptr()
    if at % 16 != 0:
        x = x.clone()
        at = x.data_ptr()
    if residual is not None:
        residual = residual.contiguous()
    call(_lib.load().mq_w4_linear, dev, at, qweight.data_ptr(), scales.data_ptr(),
         None if zeros is None else zeros.data_ptr(),
         None if residual is None else residual.data_ptr(), out.data_ptr(), x.numel() // k, n, k,
         k // groups, DTYPES[dtype], DTYPES[scales.dtype], DTYPES[out_dtype])
    return out


def _refuse(x, qweight, scales, zeros, residual, out_dtype) -> None:
    """Raises for the first of w4_linear's argument checks that fails."""
    if x.device.type != "cuda":
        raise ValueError("w4_linear expects CUDA tensors")
    if x.dtype not in _HALF:
        raise ValueError(f"w4_linear only supports fp16/bf16, got {x.dtype}")
    if out_dtype not in (None, x.dtype, torch.float32):
        raise ValueError(f"out_dtype must be {x.dtype} or float32, got {out_dtype}")
    if qweight.ndim != 2 or qweight.dtype != torch.uint8:
        raise ValueError(f"qweight must be uint8 [N, K/2], got {qweight.dtype} {tuple(qweight.shape)}")
    n, k = qweight.shape[0], 2 * qweight.shape[1]
    if x.ndim < 1 or x.shape[-1] != k:
        raise ValueError(f"x has shape {tuple(x.shape)}, the weight has K = {k}")
    if scales.ndim != 2 or scales.shape[0] != n or scales.shape[1] < 1 or k % scales.shape[1] != 0 \
            or k // scales.shape[1] not in GROUP_SIZES:
        raise ValueError(f"scales {tuple(scales.shape)} do not fit qweight {tuple(qweight.shape)} in "
                         f"groups of {GROUP_SIZES}")
    if scales.dtype not in _HALF:
        raise ValueError(f"scales must be fp16/bf16, got {scales.dtype}")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise ValueError(f"zeros must be uint8 {tuple(scales.shape)}, got {zeros.dtype} {tuple(zeros.shape)}")
    for name, t in (("qweight", qweight), ("scales", scales), ("zeros", zeros), ("residual", residual)):
        if t is not None:
            if t.device != x.device:
                raise ValueError(f"{name} is on {t.device}, x on {x.device}")
            if name != "residual" and not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
    want = (x.dtype if out_dtype is None else out_dtype, (*x.shape[:-1], n))
    raise ValueError(f"residual must be {want[0]} {want[1]}, got {residual.dtype} {tuple(residual.shape)}")
