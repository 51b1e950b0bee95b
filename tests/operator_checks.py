"""Shared by the tests of the operators around a selective state space layer: error bounds and plain forms in 64 bits.

A bound is per element: half a step of the output's type, relative to the value, plus ``ops`` roundings of fp32 relative to
``terms``, the sum of the magnitudes that were added up on the way to the value."""
import torch

F32 = 2.0 ** -24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def near(got, want, terms, ops, what="", flushed=0.0):
    """|got - want| <= half a step |want| + ops 2^-24 terms (want and terms in 64 bits) + flushed, what is lost of values that
    are too small for a normal number."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    # the smallest numbers of a type are a fixed distance apart
    floor = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bound = half_step(got.dtype) * want.abs() * (1 + 2.0 ** -6) + ops * F32 * terms + floor + flushed
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound).max()):.2f} times the bound"


def differences(f, leaves, grads, seed, step=2.0 ** -7):
    """Central differences of the scalar f(*leaves) (summed in 64 bits) along a random direction of each leaf against the
    gradients.  Rounding: f moves by at most 64 roundings of fp32 of its magnitude; the second-order remainder is taken
    from the difference between this step and twice the step (the remainder grows with its square)."""
    gen = torch.Generator(device=leaves[0].device).manual_seed(seed)
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        v = torch.randn(leaf.shape, generator=gen, device=leaf.device, dtype=leaf.dtype)

        def at(h):
            moved = [t.detach() for t in leaves]
            moved[i] = moved[i] + h * v
            total, size = f(*moved)
            return float(total), float(size)

        (a, size), (b, _), (c, _), (d, _) = at(step), at(-step), at(2 * step), at(-2 * step)
        near_, far = (a - b) / (2 * step), (c - d) / (4 * step)
        want = float((grad.double() * v.double()).sum())
        bound = 64 * F32 * size / step + abs(far - near_) + 1e-6 * float((grad.double() * v.double()).abs().sum())
        assert abs(near_ - want) <= bound, (i, near_, want, bound)


def silu(v):
    return v / (1 + torch.exp(-v))


def conv_plain(x, weight, bias, act, start):
    """short_conv of one batch in x's own type; (out, final, sum in front of the activation, sum of its magnitudes)."""
    width, tokens = weight.shape[1], x.shape[1]
    held = torch.cat([start, x], 1)
    pre = sum(held[:, k:k + tokens] * weight[:, k] for k in range(width))
    size = sum((held[:, k:k + tokens] * weight[:, k]).abs() for k in range(width))
    if bias is not None:
        pre, size = pre + bias, size + bias.abs()
    return (silu(pre) if act else pre), held[:, tokens:], pre, size


def norm_plain(x, weight, residual, eps):
    stream = x if residual is None else x + residual
    rstd = 1 / torch.sqrt(stream.square().mean(-1, keepdim=True) + eps)
    return stream * rstd * weight, stream, rstd


def scan_plain(x, dt, A, B, C, D, z, dt_bias, softplus, start):
    """selective_scan of one batch, token by token in x's own type; (out, final)."""
    per = x.shape[2] // B.shape[2]
    B, C = (t.repeat_interleave(per, 2) for t in (B, C))
    step = dt if dt_bias is None else dt + dt_bias
    if softplus:
        step = torch.logaddexp(step, torch.zeros_like(step))
    h = x.new_zeros(x.shape[0], *A.shape) if start is None else start
    y = []
    for t in range(x.shape[1]):
        h = torch.exp(step[:, t, :, None] * A) * h + (step[:, t] * x[:, t])[..., None] * B[:, t]
        y.append((h * C[:, t]).sum(-1))
    y = torch.stack(y, 1)
    if D is not None:
        y = y + D * x
    return (y if z is None else y * silu(z)), h
