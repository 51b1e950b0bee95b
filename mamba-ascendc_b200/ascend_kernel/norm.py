"""Root-mean-square norm with the residual's addition, for training and, with an output in 8 bits, for serving.

    stream = x + residual ;  out = stream / sqrt(mean(stream^2) + eps) * weight

The norm in front of every block of a Mamba network (mamba_torch/vmamba2_network.py:197-302 applies it with framework
calls); one pass over the data each way (``ssd_rms_norm_fwd``, ``ssd_rms_norm_bwd``).  Rows are normed in fp32, before the
sum is rounded to the residual's type.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _capi
from ._operands import DTYPES, activation, exactly, fail, parameter, without_gradients
from .mamba2 import _device_guard, _ptr, _requires_grad, _stream

MAX_WIDTH = 16384


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[rows, width] with the columns side by side; a view wherever the rows lie at one distance."""
    return t.reshape(-1, t.shape[-1])


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


def _args(x, weight, residual, eps: float) -> "_capi.SsdNormArgs":
    a = _capi.SsdNormArgs(x.data_ptr(), _ptr(residual), weight.data_ptr())
    a.rows, a.width = x.shape
    a.x_stride = x.stride(0)
    a.residual_stride = 0 if residual is None else residual.stride(0)
    a.dtype = DTYPES[x.dtype]
    a.residual_f32 = residual is not None and residual.dtype is torch.float32
    a.weight_f32 = weight.dtype is torch.float32
    a.eps = eps
    return a


def _forward(x, weight, residual, eps: float, want_rstd: bool):
    """(out, stream or None, rstd or None) of rows."""
    out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    stream = None if residual is None else torch.empty(x.shape, device=x.device, dtype=residual.dtype)
    rstd = torch.empty(x.shape[0], device=x.device, dtype=torch.float32) if want_rstd else None
    a = _args(x, weight, residual, eps)
    a.out, a.stream, a.rstd = out.data_ptr(), _ptr(stream), _ptr(rstd)
    with _device_guard(x.device):
        _capi.check(_capi.lib.ssd_rms_norm_fwd(ctypes.byref(a), _stream()), "rms_norm")
    return out, stream, rstd


class _RmsNorm(torch.autograd.Function):
    """Keeps the row's 1 / rms and what its sum is formed of: the fp32 stream, or x and a residual in fewer bits (the stream
    is rounded then, and the gradient of the weight would carry that rounding)."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        out, stream, rstd = _forward(x, weight, residual, eps, True)
        ctx.residual_type = None if residual is None else residual.dtype
        if residual is None:
            ctx.save_for_backward(weight, rstd, x, None)
        elif residual.dtype is torch.float32:
            ctx.save_for_backward(weight, rstd, stream, None)
        else:
            ctx.save_for_backward(weight, rstd, residual, x)
        ctx.x_type = x.dtype
        return out, stream

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dstream):
        weight, rstd, stream, addend = ctx.saved_tensors
        if dout is None and dstream is None:
            return None, None, None, None
        dout = stream.new_zeros(stream.shape, dtype=ctx.x_type) if dout is None else _side_by_side(dout)
        dstream = None if dstream is None else _side_by_side(dstream)
        rows, width = stream.shape
        want_x, want_weight, want_residual, _ = ctx.needs_input_grad
        dx = torch.empty(rows, width, device=dout.device, dtype=ctx.x_type)
        other = ctx.residual_type is not None and ctx.residual_type is not ctx.x_type and want_residual
        dresidual = torch.empty(rows, width, device=dout.device, dtype=ctx.residual_type) if other else None
        dweight = torch.empty_like(weight) if want_weight else None
        dtype = DTYPES[ctx.x_type]
        lib = _capi.lib
        with _device_guard(dout.device):
            work = (torch.empty(lib.ssd_rms_norm_work_bytes(rows, width, dtype), device=dout.device, dtype=torch.uint8)
                    if want_weight else None)
            a = _capi.SsdNormGradArgs(dout.data_ptr(), _ptr(dstream), stream.data_ptr(), _ptr(addend), weight.data_ptr(),
                                      rstd.data_ptr(), dx.data_ptr(), _ptr(dresidual), _ptr(dweight), _ptr(work), rows,
                                      dout.stride(0), 0 if dstream is None else dstream.stride(0), stream.stride(0),
                                      0 if addend is None else addend.stride(0), width, dtype,
                                      stream.dtype is torch.float32, weight.dtype is torch.float32)
            _capi.check(lib.ssd_rms_norm_bwd(ctypes.byref(a), _stream()), "rms_norm")
        if not want_residual:
            dresidual = None
        elif not other:
            dresidual = dx  # one tensor for both, as the gradient of an addition is
        return dx if want_x else None, dweight, dresidual, None


def _side_by_side(t: torch.Tensor) -> torch.Tensor:
    """A gradient may come broadcast."""
    return t if t.stride(-1) == 1 else t.contiguous()


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-5
             ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``out`` [..., width] of the norm of x, or (``out``, ``stream``) of the norm of ``stream = x + residual``.

    x [..., width] in fp32, bf16 or fp16, rows at any distance; weight [width] and residual [..., width] in fp32 or the type
    of x.  ``out`` has the type of x, ``stream`` that of the residual.  With gradients for x, weight and residual."""
    op = "rms_norm"
    _check(op, x, weight, residual)
    if x.numel() == 0:
        stream = None if residual is None else residual + x.to(residual.dtype)
        out = (x if residual is None else stream.to(x.dtype)) * weight.to(x.dtype)
        return out if residual is None else (out, stream)
    rows, extra = _rows(x), None if residual is None else _rows(residual)
    if _requires_grad(x, weight, residual):
        out, stream = _RmsNorm.apply(rows, weight, extra, float(eps))
    else:
        out, stream, _ = _forward(rows, weight, extra, float(eps), False)
    return out.view(x.shape) if residual is None else (out.view(x.shape), stream.view(x.shape))


def rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-5,
                   group_size: Optional[int] = None, scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, ...]:
    """(``q``, ``scales``) or, with a residual, (``q``, ``scales``, ``stream``): the norm as e4m3 values, ``out = q * scales``.

    ``group_size`` None: a scale per row, ``scales`` [..., 1]; 32, 64 or 128 columns that divide the width: a scale for each,
    ``scales`` [..., width / group_size].  A scale is the largest magnitude / 448, or 1 where that is 0.  ``scale`` (fp32, one
    element on the device): that one scale for everything, magnitudes above 448 cut off; it is returned as ``scales``.
    Without gradients."""
    op = "rms_norm_quant"
    _check(op, x, weight, residual)
    without_gradients(op, x, weight, residual)
    width = x.shape[-1]
    if group_size is not None and (group_size not in (32, 64, 128) or width % group_size):
        fail(op, "group_size must be 32, 64 or 128 and divide the width")
    if scale is not None:
        if group_size is not None:
            fail(op, "group_size and scale exclude each other")
        if scale.dtype is not torch.float32 or scale.numel() != 1:
            fail(op, "scale must be one float32 element")
        exactly(op, scale, "scale", tuple(scale.shape), x)
    columns = width // group_size if group_size else 1
    q = torch.empty(x.shape, device=x.device, dtype=torch.float8_e4m3fn)
    scales = scale if scale is not None else torch.empty(*x.shape[:-1], columns, device=x.device, dtype=torch.float32)
    stream = None if residual is None else torch.empty(x.shape, device=x.device, dtype=residual.dtype)
    if x.numel():
        a = _args(_rows(x), weight, None if residual is None else _rows(residual), float(eps))
        a.q, a.stream, a.group = q.data_ptr(), _ptr(stream), group_size or 0
        if scale is None:
            a.scales = scales.data_ptr()
        else:
            a.static_scale = scale.data_ptr()
        with _device_guard(x.device):
            _capi.check(_capi.lib.ssd_rms_norm_fwd(ctypes.byref(a), _stream()), op)
    return (q, scales) if residual is None else (q, scales, stream)
