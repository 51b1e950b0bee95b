"""The operators through the C ABI with the records of the ctypes binding: the bits that the Python calls return."""
import ctypes

import pytest
import torch

import ascend_kernel as ak
from ascend_kernel import _capi

pytestmark = pytest.mark.gpu

lib = _capi.lib
KINDS = {torch.float32: _capi.SSD_F32, torch.bfloat16: _capi.SSD_BF16, torch.float16: _capi.SSD_F16}


def rnd(*shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda").to(dtype)


def record(kind, **fields):
    r = kind()
    r.held = fields  # tensors stay until the call
    for name, value in fields.items():
        if isinstance(value, torch.Tensor):
            value = value.data_ptr()
        if isinstance(value, (tuple, list)):
            value = type(getattr(r, name))(*value)
        setattr(r, name, value)
    return r


def call(function, r):
    _capi.check(getattr(lib, function)(ctypes.byref(r), torch.cuda.current_stream().cuda_stream), function)


def bytes_of(count):
    return torch.empty(max(count, 1), device="cuda", dtype=torch.uint8)


@pytest.mark.parametrize("dtype", KINDS)
def test_norm(dtype):
    rows, width = 37, 200
    x, residual, weight = rnd(rows, width + 8, dtype=dtype)[:, :width], rnd(rows, width), rnd(width)
    leaves = [t.detach().requires_grad_(True) for t in (x, weight, residual)]
    out, stream = ak.rms_norm(*leaves, eps=1e-4)
    dout, dstream = torch.randn_like(out), torch.randn_like(stream)
    want = [out, stream, *torch.autograd.grad([out, stream], leaves, [dout, dstream])]
    out, stream, rstd = torch.empty_like(out), torch.empty_like(stream), torch.empty(rows, device="cuda")
    kind = dict(width=width, dtype=KINDS[dtype], residual_f32=1, weight_f32=1)
    call("ssd_rms_norm_fwd", record(_capi.SsdNormArgs, x=x, residual=residual, weight=weight, out=out, stream=stream, rstd=rstd, rows=rows,
                                    x_stride=width + 8, residual_stride=width, eps=1e-4, **kind))
    dx, dresidual, dweight = torch.empty_like(out), torch.empty_like(residual), torch.empty_like(weight)
    call("ssd_rms_norm_bwd", record(_capi.SsdNormGradArgs, dout=dout, dstream=dstream, stream=stream, weight=weight, rstd=rstd, dx=dx,
                                    dresidual=dresidual, dweight=dweight, rows=rows, dout_stride=width, dstream_stride=width,
                                    stream_stride=width, work=bytes_of(lib.ssd_rms_norm_work_bytes(rows, width, KINDS[dtype])), **kind))
    assert all(torch.equal(a, b) for a, b in zip(want, (out, stream, dx, dweight, dresidual)))
    for group, scale in ((0, None), (0, torch.tensor([0.01], device="cuda"))):
        want = ak.rms_norm_quant(x, weight, residual, 1e-4, group or None, scale)
        q, scales = torch.empty_like(want[0]), torch.empty_like(want[1])
        call("ssd_rms_norm_fwd", record(_capi.SsdNormArgs, x=x, residual=residual, weight=weight, stream=stream, q=q, rows=rows, x_stride=width + 8,
                                        residual_stride=width, eps=1e-4, group=group,
                                        **(dict(scales=scales) if scale is None else dict(static_scale=scale)), **kind))
        assert torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and (scale is not None or torch.equal(scales, want[1]))


@pytest.mark.parametrize("dtype", KINDS)
def test_convolution(dtype):
    b, l, c, w = 2, 70, 24, 3
    x, weight, bias, initial = rnd(b, l, c + 8, dtype=dtype)[..., 8:], rnd(c, w), rnd(c), rnd(b, w - 1, c, dtype=dtype)
    leaves = [t.detach().requires_grad_(True) for t in (x, weight, bias, initial)]
    out, final = ak.short_conv(*leaves[:3], "silu", leaves[3], return_final_state=True)
    dout, dfinal = torch.randn_like(out), torch.randn_like(final)
    want = [out, final, *torch.autograd.grad([out, final], leaves, [dout, dfinal])]
    out, final = torch.empty_like(out), torch.empty_like(final)
    kind = dict(channels=c, width=w, dtype=KINDS[dtype], weight_f32=1, silu=1)
    r = record(_capi.SsdConvArgs, x=x, weight=weight, bias=bias, initial_state=initial, out=out, final_state=final, tokens=l, rows=b,
               batch_stride=l * (c + 8), token_stride=c + 8, **kind)
    call("ssd_short_conv_fwd", r)
    dx, dinitial, dweight, dbias = torch.empty_like(out), torch.empty_like(initial), torch.empty_like(weight), torch.empty_like(bias)
    call("ssd_short_conv_bwd", record(_capi.SsdConvGradArgs, forward=r, dout=dout, dfinal=dfinal, dx=dx, dinitial=dinitial, dweight=dweight,
                                      dbias=dbias, work=bytes_of(lib.ssd_short_conv_work_bytes(ctypes.byref(r)))))
    assert all(torch.equal(a, b) for a, b in zip(want, (out, final, dx, dweight, dbias, dinitial)))
    token, slots, cache = rnd(b, c, dtype=dtype), torch.tensor([4, 1], device="cuda", dtype=torch.int32), rnd(6, w - 1, c, dtype=dtype)
    moved, other, out = cache.clone(), cache.clone(), torch.empty(b, c, device="cuda", dtype=dtype)
    want = ak.short_conv_step(token, moved, weight, bias, "silu", slots)
    call("ssd_short_conv_step", record(_capi.SsdConvStepArgs, x=token, weight=weight, bias=bias, state=cache, slots=slots, state_out=other, out=out,
                                       x_stride=c, state_stride=(w - 1) * c, state_out_stride=(w - 1) * c, rows=b, slot_count=6, **kind))
    assert torch.equal(out, want) and torch.equal(other, moved)


@pytest.mark.parametrize("dtype", KINDS)
def test_scan(dtype):
    b, l, c, n, g = 2, 150, 24, 8, 2
    act = lambda *s: rnd(b, l, *s, dtype=dtype)  # noqa: E731
    x, dt, z, B, C = act(c), act(c), act(c), act(g, n), act(g, n)
    A, D, bias, initial = -rnd(c, n).abs(), rnd(c), rnd(c), rnd(b, c, n)
    leaves = [t.requires_grad_(True) for t in (x, dt, A, B, C, D, z, bias, initial)]
    out, final = ak.selective_scan(*leaves[:8], True, leaves[8], return_final_state=True)
    dout, dfinal = torch.randn_like(out), torch.randn_like(final)
    want = [out, final, *torch.autograd.grad([out, final], leaves, [dout, dfinal])]
    out, final = torch.empty_like(out), torch.empty_like(final)
    kind = dict(channels=c, dstate=n, groups=g, dtype=KINDS[dtype], softplus=1)
    rows, shared = (l * c, c), (l * g * n, g * n, n)
    r = record(_capi.SsdScanArgs, x=x, dt=dt, z=z, bm=B, cm=C, A=A, D=D, dt_bias=bias, initial_state=initial, out=out, final_state=final,
               tokens=l, rows=b, x_strides=rows, dt_strides=rows, z_strides=rows, b_strides=shared, c_strides=shared, **kind)
    work = bytes_of(lib.ssd_selective_scan_work_bytes(ctypes.byref(r)))
    kept = bytes_of(lib.ssd_selective_scan_checkpoint_bytes(ctypes.byref(r)))
    r.work, r.checkpoints = work.data_ptr(), kept.data_ptr()
    call("ssd_selective_scan_fwd", r)
    grads = [torch.empty_like(t) for t in leaves]
    names = ("dx", "ddt", "dA", "dbm", "dcm", "dD", "dz", "d_dt_bias", "dinitial")
    call("ssd_selective_scan_bwd", record(_capi.SsdScanGradArgs, forward=r, dout=dout, dfinal=dfinal, **dict(zip(names, grads)),
                                          work=bytes_of(lib.ssd_selective_scan_grad_work_bytes(ctypes.byref(r)))))
    for name, a, v in zip(("out", "final") + names, [out, final, *grads], want):
        assert torch.equal(a, v), name
    x, dt, z, B, C = (t[:, 0].detach().contiguous() for t in (x, dt, z, B, C))
    A, D, bias = (t.detach() for t in (A, D, bias))
    slots, cache = torch.tensor([4, 1], device="cuda", dtype=torch.int32), rnd(6, c, n)
    moved, other, out = cache.clone(), cache.clone(), torch.empty(b, c, device="cuda", dtype=dtype)
    want = ak.selective_scan_step(x, dt, A, B, C, moved, D, z, bias, True, slots)
    call("ssd_selective_scan_step", record(_capi.SsdScanStepArgs, x=x, dt=dt, z=z, bm=B, cm=C, A=A, D=D, dt_bias=bias, state=cache, slots=slots,
                                           state_out=other, out=out, x_stride=c, dt_stride=c, z_stride=c, b_strides=(g * n, n),
                                           c_strides=(g * n, n), state_stride=c * n, state_out_stride=c * n, rows=b, slot_count=6, **kind))
    assert torch.equal(out, want) and torch.equal(other, moved)
