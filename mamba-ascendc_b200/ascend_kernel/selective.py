"""Selective scan: the state space recurrence with a decay of its own for every channel and state column (Mamba-1), beside
the SSD of ``mamba2_ssd_fwd``, whose decay is one number per head.  For prompts and training (batches and packed sequences,
initial and final states) and for generation steps of one token.

    h_t[c,n] = exp(dt_t[c] A[c,n]) h_{t-1}[c,n] + dt_t[c] x_t[c] B_t[g,n]
    out_t[c] = (sum_n C_t[g,n] h_t[c,n] + D[c] x_t[c]) * silu(z_t[c])          g = c // (channels / groups)

Names and meaning of the arguments follow ``mamba2_ssd_fwd`` (ascend_kernel/mamba2.py:1923-2017); activations may be fp32,
bf16 or fp16, parameters and states are fp32.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _capi
from ._operands import DTYPES, activation, cache, exactly, fail, packing, parameter, slot_numbers, without_gradients
from .mamba2 import _device_guard, _ptr, _requires_grad, _stream

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


def _args(x, dt, A, B, C, D, z, dt_bias, softplus: bool, initial, cu_seqlens) -> "_capi.SsdScanArgs":
    batch, tokens, channels = x.shape
    two, three = _capi._I64 * 2, _capi._I64 * 3
    rows = batch if cu_seqlens is None else cu_seqlens.numel() - 1
    return _capi.SsdScanArgs(x.data_ptr(), dt.data_ptr(), _ptr(z), B.data_ptr(), C.data_ptr(), A.data_ptr(), _ptr(D),
                             _ptr(dt_bias), _ptr(initial), _ptr(cu_seqlens), None, None, None, None, tokens,
                             two(*x.stride()[:2]), two(*dt.stride()[:2]), two(*(z.stride()[:2] if z is not None else (0, 0))),
                             three(*B.stride()[:3]), three(*C.stride()[:3]), rows, channels, A.shape[1], B.shape[2],
                             DTYPES[x.dtype], softplus)


def _floats(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes // 4, device=device, dtype=torch.float32) if nbytes else None


def _forward(x, dt, A, B, C, D, z, dt_bias, softplus, initial, cu_seqlens, want_final: bool, want_checkpoints: bool):
    out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    a = _args(x, dt, A, B, C, D, z, dt_bias, softplus, initial, cu_seqlens)
    final = torch.empty(a.rows, a.channels, a.dstate, device=x.device, dtype=torch.float32) if want_final else None
    lib, checkpoints = _capi.lib, None
    with _device_guard(x.device):
        p = ctypes.byref(a)
        if want_checkpoints:
            checkpoints = _floats(lib.ssd_selective_scan_checkpoint_bytes(p), x.device)
        work = _floats(lib.ssd_selective_scan_work_bytes(p), x.device)
        a.out, a.final_state, a.checkpoints, a.work = out.data_ptr(), _ptr(final), _ptr(checkpoints), _ptr(work)
        _capi.check(lib.ssd_selective_scan_fwd(p, _stream()), "selective_scan")
    return out, final, checkpoints


class _SelectiveScan(torch.autograd.Function):
    """Keeps its inputs and the states at every 64th token; backward forms what lies between again."""

    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, initial, softplus, cu_seqlens, want_final):
        ctx.set_materialize_grads(False)
        out, final, checkpoints = _forward(x, dt, A, B, C, D, z, dt_bias, softplus, initial, cu_seqlens, want_final, True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, initial, cu_seqlens, checkpoints)
        ctx.softplus = softplus
        return out, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dfinal):
        x, dt, A, B, C, D, z, dt_bias, initial, cu_seqlens, checkpoints = ctx.saved_tensors
        if dout is None and dfinal is None:
            return (None,) * 12
        dev = x.device
        dout = torch.zeros(x.shape, device=dev, dtype=x.dtype) if dout is None else dout.contiguous()
        dfinal = None if dfinal is None else dfinal.contiguous()
        a = _args(x, dt, A, B, C, D, z, dt_bias, ctx.softplus, initial, cu_seqlens)
        a.checkpoints = _ptr(checkpoints)

        def like(t):
            return None if t is None else torch.empty(t.shape, device=dev, dtype=t.dtype)

        dx, ddt, dz, dB, dC = like(x), like(dt), like(z), like(B), like(C)
        dA, dD, dbias = like(A), like(D), like(dt_bias)
        dinitial = like(initial) if ctx.needs_input_grad[8] else None
        lib = _capi.lib
        with _device_guard(dev):
            work = _floats(lib.ssd_selective_scan_grad_work_bytes(ctypes.byref(a)), dev)
            g = _capi.SsdScanGradArgs(a, dout.data_ptr(), _ptr(dfinal), dx.data_ptr(), ddt.data_ptr(), _ptr(dz), dB.data_ptr(),
                                      dC.data_ptr(), dA.data_ptr(), _ptr(dD), _ptr(dbias), _ptr(dinitial), _ptr(work))
            _capi.check(lib.ssd_selective_scan_bwd(ctypes.byref(g), _stream()), "selective_scan")
        grads = (dx, ddt, dA, dB, dC, dD, dz, dbias, dinitial)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None)


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
    op = "selective_scan"
    _check(op, 2, x, dt, A, B, C, D, z, dt_bias)
    rows = x.shape[0] if cu_seqlens is None else packing(op, cu_seqlens, x)
    if initial_states is not None:
        parameter(op, initial_states, "initial_states", (rows, x.shape[2], A.shape[1]), x, f32_only=True)
    if x.numel() == 0 and (cu_seqlens is None or x.shape[2] == 0):  # no tokens: the states pass through
        final = (torch.zeros(rows, x.shape[2], A.shape[1], device=x.device) if initial_states is None
                 else initial_states.clone())
        return (x.clone(), final) if return_final_state else x.clone()
    if _requires_grad(x, dt, A, B, C, D, z, dt_bias, initial_states):
        out, final = _SelectiveScan.apply(x, dt, A, B, C, D, z, dt_bias, initial_states, bool(dt_softplus), cu_seqlens,
                                          bool(return_final_state))
    else:
        out, final, _ = _forward(x, dt, A, B, C, D, z, dt_bias, bool(dt_softplus), initial_states, cu_seqlens,
                                 return_final_state, False)
    return (out, final) if return_final_state else out


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                        state: torch.Tensor, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                        dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False,
                        slots: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``selective_scan`` of one token of each of R sequences: ``out`` [R,C], and ``state`` [slots,C,N] is moved on by it.

    x, dt and z [R,C], B and C [R,G,N] as in ``selective_scan``; state fp32.  ``slots`` int32 [R] says which slot of ``state`` a
    row takes (None: its own).  A number below zero or behind the last slot marks a row of padding, whose output is zeros;
    a slot that several rows name takes them one after another.  ``state_out``, like ``state``: receives the new states
    instead, and slots that no row names are left as they were in either.  Slots may lie apart, as one layer's share of a
    larger cache does.  Without gradients."""
    op = "selective_scan_step"
    _check(op, 1, x, dt, A, B, C, D, z, dt_bias)
    without_gradients(op, x, dt, A, B, C, D, z, dt_bias, state)
    inner = tuple(A.shape)
    cache(op, state, "state", inner, torch.float32, x)
    if state_out is None:
        state_out = state
    else:
        cache(op, state_out, "state_out", inner, torch.float32, x)
        if state_out.shape != state.shape:
            fail(op, "state_out must have the shape of state")
    slot_numbers(op, slots, x, state)
    out = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    if x.numel() == 0 or state.shape[0] == 0:
        return out.zero_()
    two = _capi._I64 * 2
    a = _capi.SsdScanStepArgs(x.data_ptr(), dt.data_ptr(), _ptr(z), B.data_ptr(), C.data_ptr(), A.data_ptr(), _ptr(D),
                              _ptr(dt_bias), state.data_ptr(), _ptr(slots), state_out.data_ptr(), out.data_ptr(), x.stride(0),
                              dt.stride(0), 0 if z is None else z.stride(0), two(*B.stride()[:2]), two(*C.stride()[:2]),
                              state.stride(0), state_out.stride(0), x.shape[0], state.shape[0], x.shape[1], A.shape[1],
                              B.shape[1], DTYPES[x.dtype], bool(dt_softplus))
    with _device_guard(x.device):
        _capi.check(_capi.lib.ssd_selective_scan_step(ctypes.byref(a), _stream()), op)
    return out
