"""Selective scan: the state space recurrence with a decay of its own for every channel and state column (Mamba-1), beside
the SSD of ``mamba2_ssd_fwd``, whose decay is one number per head.  For prompts and training (batches and packed sequences,
initial and final states) and for generation steps of one token.

    h_t[c,n] = exp(dt_t[c] A[c,n]) h_{t-1}[c,n] + dt_t[c] x_t[c] B_t[g,n]
    out_t[c] = (sum_n C_t[g,n] h_t[c,n] + D[c] x_t[c]) * silu(z_t[c])          g = c // (channels / groups)

Names and meaning of the arguments follow ``mamba2_ssd_fwd`` (ascend_kernel/mamba2.py:1923-2017); activations may be fp32,
bf16 or fp16, parameters and states are fp32.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from ._capi import calls
from ._operands import (activation, apart, cache, fail, packing, parameter, slot_numbers, underived, unsupported,
                        without_gradients)

MAX_STATE = 128


def _check(op: str, lead: int, x, dt, A, B, C, D, z, dt_bias) -> None:
    """``lead``: dimensions in front of the channels (2 for [B,L,...], 1 for [R,...])."""
    names = "B,L" if lead == 2 else "R"
    activation(op, x, "x")
    if x.dim() != lead + 1:
        fail(op, f"x must have shape [{names},C]")
    for t, name in ((dt, "dt"), (z, "z"), (B, "B"), (C, "C")):
        if t is not None:
            activation(op, t, name, x)
    for t, name in ((dt, "dt"), (z, "z")):
        if t is not None and t.shape != x.shape:
            fail(op, f"{name} must have the shape of x")
    if B.dim() != lead + 2 or B.shape != C.shape or B.shape[:lead] != x.shape[:lead]:
        fail(op, f"B and C must have shape [{names},G,N]")
    channels, groups, n = x.shape[-1], B.shape[-2], B.shape[-1]
    if groups == 0 or channels % groups:
        fail(op, "channels must be divisible by groups")
    if not 0 < n <= MAX_STATE:
        fail(op, f"state size must be 1 to {MAX_STATE}")
    parameter(op, A, "A", (channels, n), x, f32_only=True)
    if D is not None:
        parameter(op, D, "D", (channels,), x, f32_only=True)
    if dt_bias is not None:
        parameter(op, dt_bias, "dt_bias", (channels,), x, f32_only=True)


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                   dt_softplus: bool = False, initial_states: Optional[torch.Tensor] = None,
                   cu_seqlens: Optional[torch.Tensor] = None, return_final_state: bool = False
                   ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``out`` [B,L,C] and, with ``return_final_state``, the state [B,C,N] behind the last token.

    x, dt and z [B,L,C], B and C [B,L,G,N] with channel c reading group c // (C/G), all of one type (fp32, bf16, fp16), their
    last dimension contiguous and the others at any distance; fp32 and contiguous: A [C,N] (the negative decay value, not
    its log), D and dt_bias [C], initial_states [B,C,N].  N up to 128.

    ``cu_seqlens`` int32 [S + 1]: the tensors [1,T,...] hold S sequences one behind another, sequence s the tokens
    cu_seqlens[s] up to cu_seqlens[s + 1], from 0 and not descending; states are [S,C,N].  Outputs of tokens behind the last
    sequence are zeros.  With gradients for every tensor but cu_seqlens."""
    got = calls.selective_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_states, cu_seqlens, return_final_state)
    if got is not None:
        return got
    op = "selective_scan"
    underived(op, x, dt, A, B, C, D, z, dt_bias, initial_states, cu_seqlens)
    _check(op, 2, x, dt, A, B, C, D, z, dt_bias)
    rows = x.shape[0] if cu_seqlens is None else packing(op, cu_seqlens, x)
    if initial_states is not None:
        parameter(op, initial_states, "initial_states", (rows, x.shape[2], A.shape[1]), x, f32_only=True)
    unsupported(op)


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                        state: torch.Tensor, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False,
                        slots: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``selective_scan`` of one token of each of R sequences: ``out`` [R,C], and ``state`` [slots,C,N] is moved on by it.

    x, dt and z [R,C], B and C [R,G,N] as in ``selective_scan``; state fp32.  ``slots`` int32 [R] says which slot of ``state`` a
    row takes (None: its own).  A number below zero or behind the last slot marks a row of padding, whose output is zeros;
    a slot that several rows name takes them one after another.  ``state_out``, like ``state``: receives the new states
    instead, and slots that no row names are left as they were in either; it may be ``state``, but no slot of it may lie on
    another one of ``state``.  Slots may lie apart, as one layer's share of a
    larger cache does.  Without gradients; what is written counts as changed in place for autograd."""
    got = calls.selective_scan_step(x, dt, A, B, C, state, D, z, dt_bias, dt_softplus, slots, state_out)
    if got is not None:
        return got
    op = "selective_scan_step"
    underived(op, x, dt, A, B, C, state, D, z, dt_bias, slots, state_out)
    _check(op, 1, x, dt, A, B, C, D, z, dt_bias)
    without_gradients(op, x, dt, A, B, C, D, z, dt_bias, state, state_out)
    inner = tuple(A.shape)
    cache(op, state, "state", inner, torch.float32, x)
    if state_out is not None:
        cache(op, state_out, "state_out", inner, torch.float32, x)
        if state_out.shape != state.shape:
            fail(op, "state_out must have the shape of state")
        apart(op, state, state_out)
    slot_numbers(op, slots, x, state)
    unsupported(op)
