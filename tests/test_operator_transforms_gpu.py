"""Forward-mode derivatives and function transforms: the operators have neither, and say so instead of returning a result whose
derivative is lost."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

import ascend_kernel as ak

pytestmark = pytest.mark.gpu

C, W, N = 24, 4, 8


def rnd(*shape):
    return torch.randn(*shape, device="cuda")


def calls():
    """(name, call, tensors) of every operator."""
    x, weight, bias = rnd(2, 9, C), rnd(C, W), rnd(C)
    A, B = -rnd(C, N).abs(), rnd(2, 9, 1, N)
    token, b = rnd(2, C), rnd(2, 1, N)
    return [
        ("short_conv", lambda x, w, b, s: ak.short_conv(x, w, b, "silu", s), [x, weight, bias, rnd(2, W - 1, C)]),
        ("short_conv_step", lambda x, s, w, b, o: ak.short_conv_step(x, s, w, b, "silu", None, o),
         [token, rnd(2, W - 1, C), weight, bias, rnd(2, W - 1, C)]),
        ("selective_scan", lambda x, dt, A, B, C_, D, z, bias, s: ak.selective_scan(x, dt, A, B, C_, D, z, bias, True, s),
         [x, rnd(2, 9, C), A, B, rnd(2, 9, 1, N), bias, rnd(2, 9, C), rnd(C), rnd(2, C, N)]),
        ("selective_scan_step", lambda x, dt, A, B, C_, s, D, z, bias, o:
            ak.selective_scan_step(x, dt, A, B, C_, s, D, z, bias, True, None, o),
         [token, rnd(2, C), A, b, rnd(2, 1, N), rnd(2, C, N), bias, rnd(2, C), rnd(C), rnd(2, C, N)]),
        ("rms_norm", lambda x, w, r: ak.rms_norm(x, w, r), [token, bias, rnd(2, C)]),
        ("rms_norm_quant", lambda x, w, r: ak.rms_norm_quant(x, w, r), [token, bias, rnd(2, C)]),
    ]


@pytest.mark.parametrize("which", range(6))
def test_tangents_are_refused(which):
    name, call, tensors = calls()[which]
    for i in range(len(tensors)):
        with fwd.dual_level():
            duals = [fwd.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(tensors)]
            with pytest.raises(RuntimeError, match=f"{name}: has no forward-mode derivatives"):
                call(*duals)
            call(*tensors)  # at the same level without a tangent


@pytest.mark.parametrize("which", range(6))
def test_transforms_are_refused(which):
    name, call, tensors = calls()[which]
    scalar = lambda *ts: next(iter(o)) if isinstance(o := call(*ts), tuple) else o  # noqa: E731
    message = f"{name}: cannot run inside a function transform"
    for i in range(len(tensors)):
        at = lambda t: scalar(*(t if j == i else v for j, v in enumerate(tensors))).float().sum()  # noqa: E731
        with pytest.raises(RuntimeError, match=message):
            torch.func.vmap(at)(torch.stack([tensors[i]] * 2))
        with pytest.raises(RuntimeError, match=message):
            torch.func.grad(at)(tensors[i])
        with pytest.raises(RuntimeError, match=message):
            torch.func.jvp(at, (tensors[i],), (tensors[i],))
    # nothing of the call is transformed, but what it allocates would be
    with pytest.raises(RuntimeError, match="inside a function transform"):
        torch.func.grad(lambda t: (t * scalar(*tensors).float()[:1].sum()).sum())(rnd(3))


@pytest.mark.parametrize("which", [0, 2, 4])
def test_derivatives_of_the_gradients_are_refused(which):
    """An upstream gradient with a tangent, and several upstream gradients at once."""
    name, call, tensors = calls()[which]
    leaves = [t.requires_grad_(True) for t in tensors]
    out = call(*leaves)
    out = out[0] if isinstance(out, tuple) else out
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match=f"{name}: its gradients have no forward-mode derivatives"):
            torch.autograd.grad(out, leaves, fwd.make_dual(torch.ones_like(out), torch.ones_like(out)), retain_graph=True)
    with pytest.raises(RuntimeError, match="inside a function transform"):
        torch.autograd.grad(out, leaves, torch.ones(3, *out.shape, device="cuda"), is_grads_batched=True, retain_graph=True)
    torch.autograd.grad(out, leaves, torch.ones_like(out))
