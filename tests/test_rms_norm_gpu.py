"""rms_norm and rms_norm_quant against the definition in 64 bits.

Roundings of the output: the sum with the residual (1 of |x| + |residual|, times rstd w), the mean of squares (a chain of at most
width / 32 additions and 10 levels per row, halved by the root), the root (2), two products.  Gradients: the same factors,
and the mean of g unit over the row, whose roundings are relative to the mean of |g unit|."""
import pytest
import torch

import ascend_kernel as ak
from operator_checks import F32, differences, near, norm_plain

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-5


def make(rows, width, dtype, residual="same", sliced=False, param=torch.float32):
    extra = 24 if sliced else 0
    x = torch.randn(rows, width + extra, device="cuda").to(dtype)[:, :width]
    weight = (1 + 0.2 * torch.randn(width, device="cuda")).to(param)
    if residual is None:
        return x, weight, None
    kind = torch.float32 if residual == "fp32" else dtype
    return x, weight, (3 * torch.randn(rows, width + extra, device="cuda")).to(kind)[:, :width]


def roundings(width):
    return width / 64 + 20


def check_forward(out, stream, x, weight, residual):
    want, sums, rstd = norm_plain(x.double(), weight.double(), None if residual is None else residual.double(), EPS)
    size = want.abs() + (0 if residual is None else (x.double().abs() + residual.double().abs()) * rstd * weight.double().abs())
    near(out, want, size, roundings(x.shape[-1]), "out")
    if residual is not None:
        near(stream, sums, sums.abs(), 1, "stream")


SHAPES = [(1, 1), (1, 8), (3, 7), (5, 192), (2, 129), (4, 257), (33, 1024), (3, 1030), (17, 4096), (2, 4095), (2, 8192),
          (1, 16384), (2, 12001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", SHAPES + [(5000, 40), (2000, 513), (2500, 2048)])
@pytest.mark.parametrize("residual,sliced", [(None, False), ("same", True), ("fp32", False)])
def test_forward(rows, width, residual, sliced, dtype):
    x, weight, extra = make(rows, width, dtype, residual, sliced)
    got = ak.rms_norm(x, weight, extra, EPS)
    out, stream = got if residual else (got, None)
    assert out.dtype is dtype and out.is_contiguous() and (stream is None or stream.dtype is extra.dtype)
    check_forward(out, stream, x, weight, extra)


def plain_gradients(x, weight, residual, dout, dstream):
    leaves = [t.detach().double().requires_grad_(True) for t in (x, weight, residual)]
    out, stream, rstd = norm_plain(*leaves, EPS)
    grads = torch.autograd.grad([out, stream], leaves, [dout.double(), dstream.double()])
    with torch.no_grad():
        w, v = weight.double(), stream
        unit = (x.double().abs() + residual.double().abs()) * rstd
        g = dout.double().abs() * w.abs()
        dv = rstd * (g + unit * (g * unit).mean(-1, keepdim=True)) + dstream.double().abs()
        dw = (dout.double().abs() * unit).sum(0)
    return grads, (dv, dw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", SHAPES + [(1500, 136), (2400, 100)])
@pytest.mark.parametrize("residual,sliced", [("same", True), ("fp32", False)])
def test_gradients(rows, width, residual, sliced, dtype):
    x, weight, extra = make(rows, width, dtype, residual, sliced)
    leaves = [t.requires_grad_(True) for t in (x.detach(), weight, extra.detach())]
    out, stream = ak.rms_norm(*leaves, EPS)
    dout, dstream = torch.randn_like(out), torch.randn_like(stream)
    got = torch.autograd.grad([out, stream], leaves, [dout, dstream])
    want, (dv, dw) = plain_gradients(x, weight, extra, dout, dstream)
    ops = 3 * roundings(width)
    near(got[0], want[0], dv, ops, "dx")
    near(got[2], want[2], dv, ops, "dresidual")
    near(got[1], want[1], dw, ops + rows, "dweight")
    assert [g.dtype for g in got] == [t.dtype for t in leaves]


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_residual(dtype):
    x, weight, _ = make(50, 320, dtype, None, param=dtype)
    leaves = [t.requires_grad_(True) for t in (x, weight)]
    out = ak.rms_norm(*leaves, eps=EPS)
    dout = torch.randn_like(out)
    got = torch.autograd.grad(out, leaves, dout)
    zero = torch.zeros_like(x).detach()
    want, (dv, dw) = plain_gradients(x, weight, zero, dout, zero)
    near(got[0], want[0], dv, 3 * roundings(320))
    near(got[1], want[1], dw, 3 * roundings(320) + 50)
    assert got[1].dtype is dtype


def test_each_gradient_alone_and_missing_upstream():
    x, weight, extra = make(20, 96, torch.bfloat16, "fp32")
    leaves = [t.requires_grad_(True) for t in (x, weight, extra)]
    out, stream = ak.rms_norm(*leaves, EPS)
    dout, dstream = torch.randn_like(out), torch.randn_like(stream)
    every = torch.autograd.grad([out, stream], leaves, [dout, dstream], retain_graph=True)
    for i in range(3):
        alone = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        o, s = ak.rms_norm(*alone, EPS)
        assert torch.equal(torch.autograd.grad([o, s], alone[i], [dout, dstream])[0], every[i])
    dx, dw, dr = torch.autograd.grad(stream, leaves, dstream, retain_graph=True, allow_unused=True)
    assert torch.equal(dr, dstream) and torch.equal(dx, dstream.to(dx.dtype)) and not dw.any()
    broadcast = torch.autograd.grad(out.sum(), leaves[0], retain_graph=True)[0]
    assert torch.equal(broadcast, torch.autograd.grad(out, leaves[0], torch.ones_like(out))[0])


def test_gradients_against_differences():
    x, weight, extra = make(7, 48, torch.float32)
    coefficients = torch.randn(7, 48, device="cuda"), torch.randn(7, 48, device="cuda")

    def f(*leaves):
        out, stream = ak.rms_norm(*leaves, EPS)
        parts = torch.cat([(out * coefficients[0]).flatten(), (stream * coefficients[1]).flatten()]).double()
        return parts.sum(), parts.abs().sum()

    leaves = [t.requires_grad_(True) for t in (x, weight, extra)]
    out, stream = ak.rms_norm(*leaves, EPS)
    differences(f, leaves, torch.autograd.grad([out, stream], leaves, list(coefficients)), 4)


E4M3_HALF = 2.0 ** -4  # relative to the value
E4M3_SMALL = 2.0 ** -10  # half a step of the smallest numbers


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,group", [(1, 32, None), (3, 7, None), (16, 4096, None), (5, 4096, 128), (3, 4095, None),
                                              (2000, 128, 32), (9, 1088, 64), (2, 16384, 128), (1300, 2048, 64)])
@pytest.mark.parametrize("residual,sliced", [(None, True), ("same", False), ("fp32", False)])
def test_quant(rows, width, group, residual, sliced, dtype):
    x, weight, extra = make(rows, width, dtype, residual, sliced)
    q, scales, *stream = ak.rms_norm_quant(x, weight, extra, EPS, group)
    groups = width // group if group else 1
    assert q.dtype is torch.float8_e4m3fn and scales.shape == (rows, groups) and q.shape == x.shape
    want, _, rstd = norm_plain(x.double(), weight.double(), None if extra is None else extra.double(), EPS)
    size = want.abs() + (0 if extra is None else (x.double().abs() + extra.double().abs()) * rstd * weight.double().abs())
    off = roundings(width) * F32 * size
    top = want.view(rows, groups, -1).abs().amax(-1)
    near(scales, top / 448, (off / F32).view(rows, groups, -1).amax(-1) / 448 + 2 * top / 448, 1, "scales")
    s = scales.double().repeat_interleave(width // groups, 1)
    value = q.double() * s
    bound = E4M3_HALF * want.abs() * (1 + 2.0 ** -6) + (E4M3_SMALL * s) + 2 * off
    assert ((value - want).abs() <= bound).all()
    # of each group the largest magnitude comes out as 448 or, rounded down on the way, not below the step before it
    assert (q.double().view(rows, groups, -1).abs().amax(-1) == 448).all()
    if residual:
        near(stream[0], x.double() + extra.double(), (x.double() + extra.double()).abs(), 1)


def test_quant_with_one_scale_for_all():
    x, weight, _ = make(40, 256, torch.bfloat16, None)
    scale = torch.tensor(0.004, device="cuda")
    q, same = ak.rms_norm_quant(x, weight, scale=scale)
    assert same is scale
    want = norm_plain(x.double(), weight.double(), None, EPS)[0] / float(scale)
    bound = E4M3_HALF * want.abs().clamp(max=448) * (1 + 2.0 ** -6) + E4M3_SMALL + 2.0 ** -15 * want.abs()
    assert ((q.double() - want.clamp(-448, 448)).abs() <= bound).all() and want.abs().max() > 448


def test_quant_of_zeros_infinities_and_nan():
    """A row of zeros has scale 1; what is not finite stays within its row and comes out as NaN where the norm is NaN."""
    x = torch.randn(6, 128, device="cuda")
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    x[4] *= 1e-30
    weight = torch.ones(128, device="cuda")
    for group in (None, 32):
        q, scales = ak.rms_norm_quant(x, weight, eps=1e-5, group_size=group)
        assert (scales[1] == 1).all() and not q[1].float().any()
        assert q[2, 5].float().isnan() and q[3].float().isnan().all()
        assert (q[[0, 5]].float().abs().amax(-1) == 448).all() and (q[4].float().abs().amax() == 448)
    out = ak.rms_norm(x, weight)
    assert out[3].isnan().all() and out[2, 5].isnan() and not out[2, :5].any() and out[[0, 1, 4, 5]].isfinite().all()


def test_leading_dimensions_and_no_rows():
    x = torch.randn(2, 3, 5, 64, device="cuda", dtype=torch.bfloat16)
    weight = torch.ones(64, device="cuda")
    out, stream = ak.rms_norm(x, weight, x)
    assert out.shape == x.shape and torch.equal(stream, x + x)
    q, scales = ak.rms_norm_quant(x.transpose(0, 1), weight, group_size=64)
    assert q.shape == (3, 2, 5, 64) and scales.shape == (3, 2, 5, 1)
    assert torch.equal(q.float(), ak.rms_norm_quant(x.transpose(0, 1).contiguous(), weight, group_size=64)[0].float())
    assert torch.equal(ak.rms_norm(x[:, :, ::2], weight), ak.rms_norm(x[:, :, ::2].contiguous(), weight))
    empty = x[:0].requires_grad_(True)
    out, stream = ak.rms_norm(empty, weight, empty.detach())
    assert out.shape == empty.shape and torch.autograd.grad(out.sum(), empty)[0].shape == empty.shape
    assert ak.rms_norm_quant(x[:0], weight)[1].shape == (0, 3, 5, 1)


def test_repeats_bit_for_bit_and_in_a_graph():
    x, weight, extra = make(3000, 768, torch.bfloat16)

    def once():
        leaves = [t.detach().requires_grad_(True) for t in (x, weight, extra)]
        out, stream = ak.rms_norm(*leaves, EPS)
        return [out, stream, *torch.autograd.grad([out, stream], leaves, [x, extra])]

    first, second = once(), once()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    ak.rms_norm_quant(x, weight, extra, group_size=128)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = once() + [t.float() for t in ak.rms_norm_quant(x, weight, extra, group_size=128)]
    x.copy_(torch.randn_like(x))
    graph.replay()
    torch.cuda.synchronize()
    eager = once() + [t.float() for t in ak.rms_norm_quant(x, weight, extra, group_size=128)]
    assert all(torch.equal(a, b) for a, b in zip(captured, eager))
