"""Short causal convolution along the tokens, in front of a state space scan: for prompts and training (batches and packed
sequences, with the state that a later call goes on from) and for generation steps of one token.

    pre[t] = bias + sum_k weight[:, k] * in[t - (width - 1) + k] ;  out = pre, or pre * sigmoid(pre)

The depthwise conv1d of every Mamba block (mamba_torch/vmamba2_network.py:197-302), token-major like the SSD's own tensors
(``ssd_short_conv_fwd``, ``ssd_short_conv_bwd``, ``ssd_short_conv_step``).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _capi
from ._operands import (DTYPES, activation as check_activation, cache, exactly, fail, packing, parameter, slot_numbers,
                        without_gradients)
from .mamba2 import _device_guard, _ptr, _requires_grad, _stream


def _silu(op: str, name: Optional[str]) -> bool:
    if name not in (None, "silu"):
        fail(op, 'activation must be None or "silu"')
    return name is not None


def _check_filter(op: str, x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor]) -> int:
    channels = x.shape[-1]
    if weight.dim() != 2 or weight.shape[0] != channels:
        fail(op, "weight must have shape [channels, width]")
    width = weight.shape[1]
    if not 2 <= width <= 4:
        fail(op, "width must be 2, 3 or 4")
    parameter(op, weight, "weight", (channels, width), x)
    if bias is not None:
        if bias.dtype is not weight.dtype:
            fail(op, "bias must have the type of weight")
        exactly(op, bias, "bias", (channels,), x)
    return width


def _args(x, weight, bias, initial, cu_seqlens, silu: bool) -> "_capi.SsdConvArgs":
    batch, tokens, channels = x.shape
    rows = batch if cu_seqlens is None else cu_seqlens.numel() - 1
    return _capi.SsdConvArgs(x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(initial), _ptr(cu_seqlens), None, None, tokens,
                             x.stride(0), x.stride(1), rows, channels, weight.shape[1], DTYPES[x.dtype],
                             weight.dtype is torch.float32, silu)


def _forward(x, weight, bias, initial, cu_seqlens, silu: bool, want_final: bool):
    out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    a = _args(x, weight, bias, initial, cu_seqlens, silu)
    final = torch.empty(a.rows, a.width - 1, a.channels, device=x.device, dtype=x.dtype) if want_final else None
    a.out, a.final_state = out.data_ptr(), _ptr(final)
    with _device_guard(x.device):
        _capi.check(_capi.lib.ssd_short_conv_fwd(ctypes.byref(a), _stream()), "short_conv")
    return out, final


class _ShortConv(torch.autograd.Function):
    """Keeps its inputs; backward forms the sum in front of the activation again."""

    @staticmethod
    def forward(ctx, x, weight, bias, initial, cu_seqlens, silu, want_final):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, initial, cu_seqlens)
        ctx.silu = silu
        return _forward(x, weight, bias, initial, cu_seqlens, silu, want_final)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal):
        x, weight, bias, initial, cu_seqlens = ctx.saved_tensors
        none = (None,) * 7
        if dout is None and dfinal is None:
            return none
        dout = torch.zeros(x.shape, device=x.device, dtype=x.dtype) if dout is None else dout.contiguous()
        dfinal = None if dfinal is None else dfinal.contiguous()
        need_x, need_weight, need_bias, need_initial = ctx.needs_input_grad[:4]
        dx = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        dinitial = torch.empty_like(initial) if need_initial else None
        need_filter = need_weight or need_bias
        dweight = torch.empty_like(weight) if need_filter else None
        dbias = torch.empty_like(bias) if need_bias else None
        lib = _capi.lib
        with _device_guard(x.device):
            forward = _args(x, weight, bias, initial, cu_seqlens, ctx.silu)
            work = (torch.empty(lib.ssd_short_conv_work_bytes(ctypes.byref(forward)), device=x.device, dtype=torch.uint8)
                    if need_filter else None)
            g = _capi.SsdConvGradArgs(forward, dout.data_ptr(), _ptr(dfinal), dx.data_ptr(), _ptr(dinitial), _ptr(dweight),
                                      _ptr(dbias), _ptr(work))
            _capi.check(lib.ssd_short_conv_bwd(ctypes.byref(g), _stream()), "short_conv")
        return dx if need_x else None, dweight if need_weight else None, dbias, dinitial, None, None, None


def short_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
               initial_states: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None,
               return_final_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``out`` [B,L,C] and, with ``return_final_state``, the state [B, width - 1, C] that the next tokens go on from: the last
    width - 1 inputs.

    x [B,L,C] in fp32, bf16 or fp16, channels side by side, tokens at any distance (a column slice of a projection); weight
    [C, width] with width 2 to 4, tap k for the input width - 1 - k tokens back, and bias [C], both in fp32 or the type of x;
    ``activation`` None or "silu"; ``initial_states`` [B, width - 1, C] in the type of x, oldest input first (None: zeros).

    ``cu_seqlens`` int32 [S + 1]: x [1,T,C] holds S sequences one behind another, sequence s the tokens cu_seqlens[s] up to
    cu_seqlens[s + 1], from 0 and not descending; states are [S, width - 1, C].  Outputs of tokens behind the last sequence
    are zeros.  With gradients for x, weight, bias and initial_states."""
    op = "short_conv"
    check_activation(op, x, "x")
    if x.dim() != 3:
        fail(op, "x must have shape [B,L,C]")
    silu = _silu(op, activation)
    width = _check_filter(op, x, weight, bias)
    rows = x.shape[0] if cu_seqlens is None else packing(op, cu_seqlens, x)
    if initial_states is not None:
        if initial_states.dtype is not x.dtype:
            fail(op, "initial_states must have the type of x")
        exactly(op, initial_states, "initial_states", (rows, width - 1, x.shape[2]), x)
    if x.numel() == 0 and (cu_seqlens is None or x.shape[2] == 0):  # no tokens: the states pass through
        final = (x.new_zeros(rows, width - 1, x.shape[2]) if initial_states is None else initial_states.clone())
        return (x.clone(), final) if return_final_state else x.clone()
    if _requires_grad(x, weight, bias, initial_states):
        out, final = _ShortConv.apply(x, weight, bias, initial_states, cu_seqlens, silu, bool(return_final_state))
    else:
        out, final = _forward(x, weight, bias, initial_states, cu_seqlens, silu, return_final_state)
    return (out, final) if return_final_state else out


def short_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                    activation: Optional[str] = None, slots: Optional[torch.Tensor] = None,
                    state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``short_conv`` of one token of each of R sequences: ``out`` [R,C], and ``state`` [slots, width - 1, C] is moved on by it.

    x [R,C]; ``slots`` int32 [R] says which slot of ``state`` a row takes (None: its own).  A number below zero or behind the
    last slot marks a row of padding, whose output is zeros; a slot that several rows name takes them one after another.
    ``state_out``, like ``state``: receives the new states instead, and slots that no row names are left as they were in
    either.  Slots may lie apart, as one layer's share of a larger cache does.  Without gradients."""
    op = "short_conv_step"
    check_activation(op, x, "x")
    if x.dim() != 2:
        fail(op, "x must have shape [R,C]")
    silu = _silu(op, activation)
    width = _check_filter(op, x, weight, bias)
    without_gradients(op, x, state, weight, bias)
    inner = (width - 1, x.shape[1])
    cache(op, state, "state", inner, x.dtype, x)
    if state_out is None:
        state_out = state
    else:
        cache(op, state_out, "state_out", inner, x.dtype, x)
        if state_out.shape != state.shape:
            fail(op, "state_out must have the shape of state")
    slot_numbers(op, slots, x, state)
    out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    if x.numel() == 0 or state.shape[0] == 0:
        return out.zero_()
    a = _capi.SsdConvStepArgs(x.data_ptr(), weight.data_ptr(), _ptr(bias), state.data_ptr(), _ptr(slots), state_out.data_ptr(),
                              out.data_ptr(), x.stride(0), state.stride(0), state_out.stride(0), x.shape[0], state.shape[0],
                              x.shape[1], width, DTYPES[x.dtype], weight.dtype is torch.float32, silu)
    with _device_guard(x.device):
        _capi.check(_capi.lib.ssd_short_conv_step(ctypes.byref(a), _stream()), op)
    return out
