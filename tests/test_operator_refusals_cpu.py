"""What the operators around a selective state space layer refuse, before any launch and in the package's words; and the checks
of the argument records at the C ABI.  No GPU: tensors that claim to be on one take the checks up to the last."""
import ctypes
import re

import pytest
import torch

import ascend_kernel as ak
from ascend_kernel import _capi

F32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64


class Fake(torch.Tensor):
    """CPU tensor that claims to be on CUDA."""

    @property
    def is_cuda(self):
        return True


def fake(*shape, dtype=F32):
    return torch.zeros(shape, dtype=dtype).as_subclass(Fake)


def refused(match, call, *args, **kwargs):
    with pytest.raises(RuntimeError, match=re.escape(match)):
        call(*args, **kwargs)


def test_short_conv():
    x, w, b = fake(2, 5, 8), fake(8, 4), fake(8)
    f = ak.short_conv
    refused("short_conv: x must be a CUDA tensor", f, torch.zeros(2, 5, 8), torch.zeros(8, 4))
    refused("short_conv: x must be float32, bfloat16 or float16", f, fake(2, 5, 8, dtype=F64), w)
    refused("short_conv: x must have shape [B,L,C]", f, fake(5, 8), w)
    refused("short_conv: x must be contiguous in its last dimension", f, fake(2, 8, 5).transpose(1, 2), w)
    refused('short_conv: activation must be None or "silu"', f, x, w, b, "gelu")
    refused("short_conv: weight must have shape [channels, width]", f, x, fake(7, 4))
    refused("short_conv: width must be 2, 3 or 4", f, x, fake(8, 5))
    refused("short_conv: width must be 2, 3 or 4", f, x, fake(8, 1))
    refused("short_conv: weight must be float32 or have the type of x", f, x, fake(8, 4, dtype=BF16))
    refused("short_conv: weight must be contiguous", f, x, fake(4, 8).t())
    refused("short_conv: bias must have the type of weight", f, fake(2, 5, 8, dtype=BF16), w, fake(8, dtype=BF16))
    refused("short_conv: bias must have shape [8]", f, x, w, fake(9))
    refused("short_conv: initial_states must have shape [2, 3, 8]", f, x, w, b, None, fake(2, 4, 8))
    refused("short_conv: initial_states must have the type of x", f, x, w, b, None, fake(2, 3, 8, dtype=BF16))
    cu = torch.tensor([0, 5], dtype=torch.int32)
    refused("short_conv: with cu_seqlens the batch must be 1", f, x, w, cu_seqlens=cu)
    refused("short_conv: cu_seqlens must be a contiguous int32 tensor [sequences + 1]", f, x[:1], w, cu_seqlens=cu.long())
    refused("short_conv: cu_seqlens must be a contiguous int32 tensor [sequences + 1]", f, x[:1], w, cu_seqlens=cu[:1])
    refused("short_conv: initial_states must have shape [1, 3, 8]", f, x[:1], w, initial_states=fake(2, 3, 8), cu_seqlens=cu)
    # nothing wrong but that it is not on a GPU after all
    refused("short_conv: takes plain strided CUDA tensors only", f, x, w, b, "silu", fake(2, 3, 8), return_final_state=True)


def test_short_conv_step():
    x, w, state = fake(6, 8), fake(8, 4), fake(6, 3, 8)
    f = ak.short_conv_step
    refused("short_conv_step: x must be a CUDA tensor", f, torch.zeros(6, 8), state, w)
    refused("short_conv_step: x must have shape [R,C]", f, fake(6, 1, 8), state, w)
    refused("short_conv_step: state must have shape [slots, 3, 8]", f, x, fake(6, 8, 3), w)
    refused("short_conv_step: state must be bfloat16", f, fake(6, 8, dtype=BF16), state, fake(8, 4))
    refused("short_conv_step: state must be contiguous within a slot", f, x, fake(6, 8, 3).transpose(1, 2), w)
    refused("short_conv_step: state must have its slots apart", f, x, fake(1, 3, 8).expand(6, 3, 8), w)
    refused("short_conv_step: without slots the state must have a row for each row of x", f, x, fake(7, 3, 8), w)
    refused("short_conv_step: slots must be a contiguous int32 tensor", f, x, state, w, slots=torch.zeros(6))
    refused("short_conv_step: slots must be a contiguous int32 tensor", f, x, state, w, slots=torch.zeros(5, dtype=torch.int32))
    refused("short_conv_step: state_out must have the shape of state", f, x, state, w, state_out=fake(7, 3, 8))
    refused("short_conv_step: has no gradients", f, x, state, fake(8, 4).requires_grad_(True))


def test_selective_scan():
    x, A, B = fake(2, 5, 8), fake(8, 16), fake(2, 5, 2, 16)
    f = ak.selective_scan
    refused("selective_scan: x must be a CUDA tensor", f, *[torch.zeros(2, 5, 8)] * 5)
    refused("selective_scan: x must have shape [B,L,C]", f, fake(5, 8), x, A, B, B)
    refused("selective_scan: dt must have the shape of x", f, x, fake(2, 5, 9), A, B, B)
    refused("selective_scan: dt must have the type of x", f, x, fake(2, 5, 8, dtype=BF16), A, B, B)
    refused("selective_scan: z must have the shape of x", f, x, x, A, B, B, None, fake(2, 4, 8))
    refused("selective_scan: B and C must have shape [B,L,G,N]", f, x, x, A, fake(2, 5, 16), fake(2, 5, 16))
    refused("selective_scan: B and C must have shape [B,L,G,N]", f, x, x, A, B, fake(2, 5, 1, 16))
    refused("selective_scan: channels must be divisible by groups", f, x, x, A, fake(2, 5, 3, 16), fake(2, 5, 3, 16))
    refused("selective_scan: state size must be 1 to 128", f, x, x, fake(8, 129), fake(2, 5, 1, 129), fake(2, 5, 1, 129))
    refused("selective_scan: A must have shape [8, 16]", f, x, x, fake(8), B, B)
    low = fake(2, 5, 8, dtype=BF16), fake(2, 5, 2, 16, dtype=BF16)
    refused("selective_scan: A must be float32", f, low[0], low[0], fake(8, 16, dtype=BF16), low[1], low[1])
    refused("selective_scan: D must have shape [8]", f, x, x, A, B, B, fake(8, 1))
    refused("selective_scan: dt_bias must be contiguous", f, x, x, A, B, B, None, None, fake(16)[::2])
    refused("selective_scan: initial_states must have shape [2, 8, 16]", f, x, x, A, B, B, initial_states=fake(2, 16, 8))
    refused("selective_scan: with cu_seqlens the batch must be 1", f, x, x, A, B, B,
            cu_seqlens=torch.tensor([0, 5], dtype=torch.int32))


def test_selective_scan_step():
    x, A, B, state = fake(6, 8), fake(8, 16), fake(6, 1, 16), fake(9, 8, 16)
    slots = torch.zeros(6, dtype=torch.int32)
    f = ak.selective_scan_step
    refused("selective_scan_step: x must have shape [R,C]", f, fake(6, 1, 8), x, A, B, B, state)
    refused("selective_scan_step: B and C must have shape [R,G,N]", f, x, x, A, fake(6, 16), fake(6, 16), state)
    refused("selective_scan_step: without slots the state must have a row for each row of x", f, x, x, A, B, B, state)
    refused("selective_scan_step: state must be float32", f, x, x, A, B, B, fake(9, 8, 16, dtype=BF16), slots=slots)
    refused("selective_scan_step: state must have shape [slots, 8, 16]", f, x, x, A, B, B, fake(9, 16, 8), slots=slots)
    refused("selective_scan_step: state_out must be float32", f, x, x, A, B, B, state, slots=slots,
            state_out=fake(9, 8, 16, dtype=BF16))
    refused("selective_scan_step: slots must be a contiguous int32 tensor", f, x, x, A, B, B, state, slots=slots.long())
    refused("selective_scan_step: has no gradients", f, x, x, A, B, B, fake(9, 8, 16).requires_grad_(True), slots=slots)


def test_norms():
    x, w = fake(3, 96), fake(96)
    for f, op in ((ak.rms_norm, "rms_norm"), (ak.rms_norm_quant, "rms_norm_quant")):
        refused(f"{op}: x must be a CUDA tensor", f, torch.zeros(3, 96), torch.zeros(96))
        refused(f"{op}: x must be float32, bfloat16 or float16", f, fake(3, 96, dtype=F64), w)
        refused(f"{op}: x must have shape [..., width]", f, fake(), w)
        refused(f"{op}: x must be contiguous in its last dimension", f, fake(96, 3).t(), w)
        refused(f"{op}: width must be 1 to 16384", f, fake(1, 16385), fake(16385))
        refused(f"{op}: weight must have shape [96]", f, x, fake(95))
        refused(f"{op}: residual must have the shape of x", f, x, w, fake(2, 96))
        refused(f"{op}: residual must be float32 or have the type of x", f, x, w, fake(3, 96, dtype=BF16))
        refused(f"{op}: residual must be contiguous in its last dimension", f, x, w, fake(96, 3).t())
    q = ak.rms_norm_quant
    for group in (0, 16, 48, 64, 256):
        refused("rms_norm_quant: group_size must be 32, 64 or 128 and divide the width", q, x, w, group_size=group)
    refused("rms_norm_quant: group_size and scale exclude each other", q, x, w, group_size=32, scale=fake(1))
    refused("rms_norm_quant: scale must be one float32 element", q, x, w, scale=fake(2))
    refused("rms_norm_quant: has no gradients", q, x, fake(96).requires_grad_(True))


def record(kind, **fields):
    r = kind()
    for name, value in fields.items():
        setattr(r, name, value)
    return r


def code(function, r):
    return getattr(_capi.lib, function)(ctypes.byref(r) if r is not None else None, None)


def test_records_are_checked_before_any_launch():
    """Null records and pointers, sizes that are none, and sizes beyond what is covered: an error code, nothing launched."""
    null, shape, unsupported, out_of_range = -1, -2, -3, -4
    for f in ("ssd_rms_norm_fwd", "ssd_rms_norm_bwd", "ssd_short_conv_fwd", "ssd_short_conv_bwd", "ssd_short_conv_step",
              "ssd_selective_scan_fwd", "ssd_selective_scan_bwd", "ssd_selective_scan_step"):
        assert code(f, None) == null
    here = ctypes.addressof(ctypes.create_string_buffer(64))
    norm = dict(rows=2, width=64, x=here, weight=here, out=here)
    assert code("ssd_rms_norm_fwd", record(_capi.SsdNormArgs, **{**norm, "rows": 0})) == shape
    assert code("ssd_rms_norm_fwd", record(_capi.SsdNormArgs, **{**norm, "width": 16385})) == unsupported
    assert code("ssd_rms_norm_fwd", record(_capi.SsdNormArgs, **{**norm, "out": None})) == null
    assert code("ssd_rms_norm_fwd", record(_capi.SsdNormArgs, **norm, group=48)) == shape
    assert code("ssd_rms_norm_fwd", record(_capi.SsdNormArgs, **norm, dtype=3)) == unsupported
    assert code("ssd_rms_norm_bwd", record(_capi.SsdNormGradArgs, rows=2, width=64, dout=here)) == null
    conv = dict(rows=1, tokens=5, channels=8, width=4, x=here, weight=here, out=here)
    assert code("ssd_short_conv_fwd", record(_capi.SsdConvArgs, **{**conv, "width": 5})) == unsupported
    assert code("ssd_short_conv_fwd", record(_capi.SsdConvArgs, **{**conv, "tokens": 0})) == shape
    assert code("ssd_short_conv_fwd", record(_capi.SsdConvArgs, **{**conv, "tokens": 2 ** 31})) == out_of_range
    assert code("ssd_short_conv_fwd", record(_capi.SsdConvArgs, **{**conv, "x": None})) == null
    step = dict(rows=2, slot_count=1, channels=8, width=4, x=here, weight=here, state=here, state_out=here, out=here)
    assert code("ssd_short_conv_step", record(_capi.SsdConvStepArgs, **step)) == shape  # two rows, one slot
    scan = dict(rows=1, tokens=5, channels=8, dstate=16, groups=1, x=here, dt=here, bm=here, cm=here, A=here, out=here)
    assert code("ssd_selective_scan_fwd", record(_capi.SsdScanArgs, **{**scan, "dstate": 129})) == unsupported
    assert code("ssd_selective_scan_fwd", record(_capi.SsdScanArgs, **{**scan, "groups": 3})) == shape
    assert code("ssd_selective_scan_fwd", record(_capi.SsdScanArgs, **{**scan, "A": None})) == null
    wide = record(_capi.SsdScanArgs, **scan)
    wide.x_strides[1] = 2 ** 29
    assert code("ssd_selective_scan_fwd", wide) == out_of_range
    assert _capi.lib.ssd_selective_scan_work_bytes(None) == 0 and _capi.lib.ssd_short_conv_work_bytes(None) == 0
    assert _capi.lib.ssd_rms_norm_work_bytes(0, 64, 0) == 0


def test_records_have_the_headers_layout():
    """Sizes as the C compiler lays the records out: pointers and 64-bit numbers first, then 32-bit ones, padded to eight."""
    def size(pointers, wide, narrow):
        return (8 * (pointers + wide) + 4 * narrow + 7) // 8 * 8

    assert ctypes.sizeof(_capi.SsdNormArgs) == size(9, 3, 6)
    assert ctypes.sizeof(_capi.SsdNormGradArgs) == size(10, 5, 4)
    assert ctypes.sizeof(_capi.SsdConvArgs) == size(7, 3, 6)
    assert ctypes.sizeof(_capi.SsdConvGradArgs) == size(7, 3, 6) + 7 * 8
    assert ctypes.sizeof(_capi.SsdConvStepArgs) == size(7, 3, 7)
    assert ctypes.sizeof(_capi.SsdScanArgs) == size(14, 1 + 6 + 6, 6)
    assert ctypes.sizeof(_capi.SsdScanGradArgs) == size(14, 13, 6) + 12 * 8
    assert ctypes.sizeof(_capi.SsdScanStepArgs) == size(12, 3 + 4 + 2, 7)
