"""The words in which the operators refuse forward-mode derivatives and function transforms.  No GPU: tensors that claim to be on
one take the checks."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import ascend_kernel as ak
from test_operator_refusals_cpu import fake, refused

CALLS = {
    "rms_norm": (ak.rms_norm, [fake(3, 96), fake(96), fake(3, 96)]),
    "rms_norm_quant": (ak.rms_norm_quant, [fake(3, 96), fake(96), fake(3, 96)]),
    "short_conv": (ak.short_conv, [fake(2, 5, 8), fake(8, 4), fake(8)]),
    "short_conv_step": (ak.short_conv_step, [fake(2, 8), fake(2, 3, 8), fake(8, 4)]),
    "selective_scan": (ak.selective_scan, [fake(2, 5, 8), fake(2, 5, 8), fake(8, 16), fake(2, 5, 1, 16), fake(2, 5, 1, 16)]),
    "selective_scan_step": (ak.selective_scan_step, [fake(2, 8), fake(2, 8), fake(8, 16), fake(2, 1, 16), fake(2, 1, 16), fake(2, 8, 16)]),
}


@pytest.mark.parametrize("op", CALLS)
def test_tangents(op):
    call, tensors = CALLS[op]
    for i in range(len(tensors)):
        with fwd.dual_level():
            duals = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(tensors)]
            refused(f"{op}: has no forward-mode derivatives", call, *duals)
            refused(f"{op}: takes plain strided CUDA tensors only", call, *tensors)


@pytest.mark.parametrize("op", CALLS)
def test_transforms(op):
    call, tensors = CALLS[op]
    plain = [t.as_subclass(torch.Tensor) for t in tensors]
    for i in range(len(plain)):
        at = lambda t: call(*(t if j == i else v for j, v in enumerate(plain)))  # noqa: E731
        message = f"{op}: cannot run inside a function transform (vmap, grad, jvp)"
        refused(message, torch.func.vmap(at), torch.stack([plain[i]] * 2))
        refused(message, torch.func.grad(at), plain[i])
        refused(message, torch.func.jvp, at, (plain[i],), (plain[i],))
