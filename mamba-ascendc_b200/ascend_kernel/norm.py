"""Root-mean-square norm with the residual's addition, for training and, with an output in 8 bits, for serving.

    stream = x + residual ;  out = stream / sqrt(mean(stream^2) + eps) * weight

The norm in front of every block of a Mamba network; one pass over the data each way (``ssd_rms_norm_fwd``,
``ssd_rms_norm_bwd``).  Rows are normed in fp32, before the sum is rounded to the residual's type.  The reference has no such
operator; its demo network has the framework's layer norm in that place (mamba_torch/vmamba2_network.py:197-302).
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from ._capi import calls
from ._operands import activation, exactly, fail, parameter, underived, unsupported, without_gradients

MAX_WIDTH = 16384


def _check(op: str, x, weight, residual) -> None:
    if x.dim() < 1:
        fail(op, "x must have shape [..., width]")
    activation(op, x, "x")
    if not 0 < x.shape[-1] <= MAX_WIDTH:
        fail(op, f"width must be 1 to {MAX_WIDTH}")
    parameter(op, weight, "weight", (x.shape[-1],), x)
    if residual is not None:
        if residual.device != x.device:
            fail(op, "residual must be on the device of x")
        if residual.dtype is not torch.float32 and residual.dtype is not x.dtype:
            fail(op, "residual must be float32 or have the type of x")
        if residual.shape != x.shape:
            fail(op, "residual must have the shape of x")
        if residual.stride(-1) != 1 and residual.shape[-1] > 1:
            fail(op, "residual must be contiguous in its last dimension")


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-5
             ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``out`` [..., width] of the norm of x, or (``out``, ``stream``) of the norm of ``stream = x + residual``.

    x [..., width] in fp32, bf16 or fp16, rows at any distance; weight [width] and residual [..., width] in fp32 or the type
    of x.  ``out`` has the type of x, ``stream`` that of the residual.  With gradients for x, weight and residual."""
    got = calls.rms_norm(x, weight, residual, eps)
    if got is not None:
        return got
    op = "rms_norm"
    underived(op, x, weight, residual)
    _check(op, x, weight, residual)
    unsupported(op)


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-5,
                   group_size: Optional[int] = None, scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, ...]:
    """(``q``, ``scales``) or, with a residual, (``q``, ``scales``, ``stream``): the norm as e4m3 values, ``out = q * scales``.

    ``group_size`` None: a scale per row, ``scales`` [..., 1]; 32, 64 or 128 columns that divide the width: a scale for each,
    ``scales`` [..., width / group_size].  A scale is the largest magnitude / 448, or 1 where that is 0.  ``scale`` (fp32, one
    element on the device): that one scale for everything, magnitudes above 448 cut off; it is returned as ``scales``.
    Without gradients."""
    if group_size != 0:
        got = calls.rms_norm_quant(x, weight, residual, eps, group_size or 0, scale)
        if got is not None:
            return got
    op = "rms_norm_quant"
    underived(op, x, weight, residual, scale)
    _check(op, x, weight, residual)
    without_gradients(op, x, weight, residual)
    if group_size is not None and (group_size not in (32, 64, 128) or x.shape[-1] % group_size):
        fail(op, "group_size must be 32, 64 or 128 and divide the width")
    if scale is not None:
        if group_size is not None:
            fail(op, "group_size and scale exclude each other")
        if scale.dtype is not torch.float32 or scale.numel() != 1:
            fail(op, "scale must be one float32 element")
        exactly(op, scale, "scale", tuple(scale.shape), x)
    unsupported(op)
