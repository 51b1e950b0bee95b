"""Short causal convolution along the tokens, in front of a state space scan: for prompts and training (batches and packed
sequences, with the state that a later call goes on from) and for generation steps of one token.

    pre[t] = bias + sum_k weight[:, k] * in[t - (width - 1) + k] ;  out = pre, or pre * sigmoid(pre)

The depthwise conv1d of a Mamba block, token-major like the SSD's own tensors (``ssd_short_conv_fwd``, ``ssd_short_conv_bwd``,
``ssd_short_conv_step``).  The reference has no such operator; its demo network has the framework's 3x3 convolution over the
image in that place (mamba_torch/vmamba2_network.py:197-302).
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from ._capi import calls
from ._operands import (activation as check_activation, apart, cache, exactly, fail, packing, parameter, slot_numbers,
                        underived, unsupported, without_gradients)


def _silu(op: str, name: Optional[str]) -> None:
    if name not in (None, "silu"):
        fail(op, 'activation must be None or "silu"')


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
    if activation is None or activation == "silu":
        got = calls.short_conv(x, weight, bias, activation is not None, initial_states, cu_seqlens, return_final_state)
        if got is not None:
            return got
    op = "short_conv"
    underived(op, x, weight, bias, initial_states, cu_seqlens)
    check_activation(op, x, "x")
    if x.dim() != 3:
        fail(op, "x must have shape [B,L,C]")
    _silu(op, activation)
    width = _check_filter(op, x, weight, bias)
    rows = x.shape[0] if cu_seqlens is None else packing(op, cu_seqlens, x)
    if initial_states is not None:
        if initial_states.dtype is not x.dtype:
            fail(op, "initial_states must have the type of x")
        exactly(op, initial_states, "initial_states", (rows, width - 1, x.shape[2]), x)
    unsupported(op)


def short_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                    activation: Optional[str] = None, slots: Optional[torch.Tensor] = None,
                    state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``short_conv`` of one token of each of R sequences: ``out`` [R,C], and ``state`` [slots, width - 1, C] is moved on by it.

    x [R,C]; ``slots`` int32 [R] says which slot of ``state`` a row takes (None: its own).  A number below zero or behind the
    last slot marks a row of padding, whose output is zeros; a slot that several rows name takes them one after another.
    ``state_out``, like ``state``: receives the new states instead, and slots that no row names are left as they were in
    either; it may be ``state``, but no slot of it may lie on another one of ``state``.  Slots may lie apart, as one layer's
    share of a larger cache does.  Without gradients; what is written counts as changed in place for autograd."""
    if activation is None or activation == "silu":
        got = calls.short_conv_step(x, state, weight, bias, activation is not None, slots, state_out)
        if got is not None:
            return got
    op = "short_conv_step"
    underived(op, x, state, weight, bias, slots, state_out)
    check_activation(op, x, "x")
    if x.dim() != 2:
        fail(op, "x must have shape [R,C]")
    _silu(op, activation)
    width = _check_filter(op, x, weight, bias)
    without_gradients(op, x, state, weight, bias, state_out)
    inner = (width - 1, x.shape[1])
    cache(op, state, "state", inner, x.dtype, x)
    if state_out is not None:
        cache(op, state_out, "state_out", inner, x.dtype, x)
        if state_out.shape != state.shape:
            fail(op, "state_out must have the shape of state")
        apart(op, state, state_out)
    slot_numbers(op, slots, x, state)
    unsupported(op)
