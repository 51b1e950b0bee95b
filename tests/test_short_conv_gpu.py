"""short_conv and short_conv_step against the definition in 64 bits.

Roundings: the sum in front of the activation has one per tap and one for the bias (W + 1, of the sum of magnitudes); the
logistic function adds the rounding of its argument (|pre| 2^-24 each for the product and the exponent, the exponential's two
steps, the addition and the division's two): 8 (1 + |pre|) roundings of the output.  Gradients take the same factors once
more and then a sum over taps or over tokens."""
import pytest
import torch

import ascend_kernel as ak
from operator_checks import conv_plain, differences, near

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(b, l, c, w, dtype, sliced=False, start=True, param=torch.float32, states=None):
    wide = torch.randn(b, l, c + 24, device="cuda").to(dtype)
    x = wide[..., 16:16 + c] if sliced else wide[..., :c].contiguous()
    weight = (torch.randn(c, w, device="cuda") * w ** -0.5).to(param)
    bias = (0.3 * torch.randn(c, device="cuda")).to(param)
    initial = torch.randn(states or b, w - 1, c, device="cuda").to(dtype) if start else None
    return x, weight, bias, initial


def check_forward(out, final, x, weight, bias, act, initial):
    start = torch.zeros(x.shape[0], weight.shape[1] - 1, x.shape[2], device="cuda", dtype=torch.float64) \
        if initial is None else initial.double()
    want, last, pre, size = conv_plain(x.double(), weight.double(), None if bias is None else bias.double(), act, start)
    terms = 1.2 * (weight.shape[1] + 2) * size + (8 * (1 + pre.abs()) * want.abs() if act else 0)
    near(out, want, terms, 1, "out")
    if final is not None:
        assert torch.equal(final.double(), last)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,l,c,w,sliced,start", [
    (1, 1, 8, 4, False, True), (2, 2, 64, 4, False, False), (3, 3, 7, 4, False, True), (1, 37, 129, 3, True, True),
    (2, 130, 512, 4, True, False), (1, 1000, 1030, 2, False, True), (2, 65, 1792, 4, True, True), (1, 4097, 24, 4, False, True),
])
@pytest.mark.parametrize("act", [None, "silu"])
def test_forward(b, l, c, w, sliced, start, act, dtype):
    x, weight, bias, initial = make(b, l, c, w, dtype, sliced, start)
    bias = bias if c % 2 == 0 else None
    out, final = ak.short_conv(x, weight, bias, act, initial, return_final_state=True)
    assert out.dtype is dtype and final.dtype is dtype and out.is_contiguous()
    check_forward(out, final, x, weight, bias, act, initial)
    assert torch.equal(out, ak.short_conv(x, weight, bias, act, initial))


def plain_gradients(x, weight, bias, act, initial, dout, dfinal):
    """Gradients in 64 bits by the formula, and the sums of magnitudes behind them."""
    leaves = [t.detach().double().requires_grad_(True) for t in (x, weight, bias, initial)]
    out, final, pre, size = conv_plain(leaves[0], leaves[1], leaves[2], act, leaves[3])
    grads = torch.autograd.grad([out, final], leaves, [dout.double(), dfinal.double()])
    w, width, tokens = weight.double().abs(), weight.shape[1], x.shape[1]
    pre, size = pre.detach(), size.detach()
    # the derivative of the activation is below 1.1 and moves by at most half of what its argument is off
    slack = dout.double().abs() * ((1.1 * 16 * (1 + pre.abs()) + (width + 2) * size) if act else 1)
    held = torch.cat([initial, x], 1).double().abs()
    through = torch.zeros_like(held)
    for k in range(width):
        through[:, k:k + tokens] += slack * w[:, k]
    through[:, tokens:] += dfinal.double().abs()
    dw = torch.stack([(slack * held[:, k:k + tokens]).sum((0, 1)) for k in range(width)], 1)
    return grads, [through[:, width - 1:], dw, slack.sum((0, 1)), through[:, :width - 1]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,l,c,w,sliced,act", [
    (1, 1, 8, 4, False, "silu"), (2, 2, 5, 4, False, "silu"), (2, 131, 132, 4, True, "silu"), (3, 64, 520, 3, False, None),
    (1, 700, 33, 2, True, "silu"), (2, 300, 640, 4, False, "silu"),
])
def test_gradients(b, l, c, w, sliced, act, dtype):
    x, weight, bias, initial = make(b, l, c, w, dtype, sliced)
    leaves = [t.requires_grad_(True) for t in (x.detach(), weight, bias, initial)]
    out, final = ak.short_conv(*leaves[:3], act, leaves[3], return_final_state=True)
    dout, dfinal = torch.randn_like(out), torch.randn_like(final)
    got = torch.autograd.grad([out, final], leaves, [dout, dfinal])
    want, terms = plain_gradients(x, weight, bias, act, initial, dout, dfinal)
    # over taps w roundings more; over tokens one for each token that a thread, then a column, adds up
    for name, g, v, t, ops in zip(("dx", "dweight", "dbias", "dinitial"), got, want, terms,
                                  (w + 2, b * l + 2, b * l + 2, w + 2)):
        assert g.dtype in (dtype, torch.float32)
        near(g, v.detach(), t, ops, name)


def test_parameters_in_the_activations_type():
    x, weight, bias, initial = make(2, 50, 96, 4, torch.bfloat16, param=torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, weight, bias, initial)]
    out, final = ak.short_conv(*leaves[:3], "silu", leaves[3], return_final_state=True)
    check_forward(out.detach(), final.detach(), x.detach(), weight.detach(), bias.detach(), "silu", initial.detach())
    dout, dfinal = torch.randn_like(out), torch.randn_like(final)
    got = torch.autograd.grad([out, final], leaves, [dout, dfinal])
    want, terms = plain_gradients(x, weight, bias, "silu", initial, dout, dfinal)
    for g, v, t, leaf in zip(got, want, terms, leaves):
        assert g.dtype is leaf.dtype
        near(g, v.detach(), t, 102)


def test_each_gradient_alone_and_missing_upstream():
    x, weight, bias, initial = make(2, 33, 40, 4, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, weight, bias, initial)]
    out, final = ak.short_conv(*leaves[:3], "silu", leaves[3], return_final_state=True)
    upstream = torch.randn_like(out), torch.randn_like(final)
    every = torch.autograd.grad([out, final], leaves, upstream, retain_graph=True)
    for i, leaf in enumerate(leaves):
        alone = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        o, f = ak.short_conv(*alone[:3], "silu", alone[3], return_final_state=True)
        assert torch.equal(torch.autograd.grad([o, f], alone[i], upstream)[0], every[i])
    only_final = torch.autograd.grad(final, leaves, upstream[1], retain_graph=True, allow_unused=True)
    want = torch.zeros_like(x)
    want[:, -3:] = upstream[1]
    assert torch.equal(only_final[0], want) and not only_final[1].any()
    broadcast = torch.autograd.grad(out.sum(), leaves[0])[0]  # an upstream gradient with strides of zero
    assert torch.equal(broadcast, torch.autograd.grad(ak.short_conv(*leaves[:3], "silu", leaves[3]), leaves[0],
                                                      torch.ones_like(out))[0])


def test_gradients_against_differences():
    x, weight, bias, initial = make(1, 19, 12, 4, torch.float32)
    coefficients = torch.randn(1, 19, 12, device="cuda"), torch.randn(1, 3, 12, device="cuda")

    def f(*leaves):
        out, final = ak.short_conv(*leaves[:3], "silu", leaves[3], return_final_state=True)
        parts = torch.cat([(out * coefficients[0]).flatten(), (final * coefficients[1]).flatten()]).double()
        return parts.sum(), parts.abs().sum()

    leaves = [t.requires_grad_(True) for t in (x, weight, bias, initial)]
    out, final = ak.short_conv(*leaves[:3], "silu", leaves[3], return_final_state=True)
    differences(f, leaves, torch.autograd.grad([out, final], leaves, list(coefficients)), 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths,behind,c", [([5], 0, 16), ([1, 0, 2, 37, 0, 130, 3, 0], 5, 72), ([0, 0], 3, 9),
                                              ([700, 1, 1, 1, 299], 0, 136), ([2] * 300, 1, 8)])
def test_packed_sequences(lengths, behind, c, dtype):
    total, count = sum(lengths) + behind, len(lengths)
    x, weight, bias, initial = make(1, total, c, 4, dtype, sliced=True, states=count)
    cu = torch.tensor([0] + lengths).cumsum(0).to("cuda", torch.int32)
    leaves = [t.detach().requires_grad_(True) for t in (x, weight, bias, initial)]
    out, final = ak.short_conv(*leaves[:3], "silu", leaves[3], cu, True)
    dout, dfinal = torch.randn_like(out), torch.randn_like(final)
    grads = torch.autograd.grad([out, final], leaves, [dout, dfinal])
    with torch.no_grad():
        again = ak.short_conv(x, weight, bias, "silu", initial, cu, True)
    assert torch.equal(again[0], out) and torch.equal(again[1], final)
    at, sums = 0, [torch.zeros(c, 4, dtype=torch.float64, device="cuda") for _ in range(2)]
    for s, n in enumerate(lengths):
        own = slice(at, at + n)
        part = [x[:, own], weight, bias, initial[s:s + 1]]
        if n:
            check_forward(out.detach()[:, own], final.detach()[s:s + 1], *part[:3], "silu", part[3])
            want, terms = plain_gradients(*part[:3], "silu", part[3], dout[:, own], dfinal[s:s + 1])
            near(grads[0][:, own], want[0], terms[0], 6)
            near(grads[3][s:s + 1], want[3], terms[3], 6)
            sums = [sums[0] + want[1], sums[1] + terms[1]]
        else:
            assert torch.equal(final[s], initial[s]) and torch.equal(grads[3][s], dfinal[s])
        at += n
    near(grads[1], sums[0], sums[1], total + 2)
    assert not out[:, at:].any() and not grads[0][:, at:].any()


def test_no_tokens():
    x, weight, bias, initial = make(2, 0, 16, 4, torch.float32)
    out, final = ak.short_conv(x, weight, bias, "silu", initial, return_final_state=True)
    assert out.shape == (2, 0, 16) and torch.equal(final, initial)
    initial.requires_grad_(True)
    _, final = ak.short_conv(x, weight, bias, "silu", initial, return_final_state=True)
    assert torch.equal(torch.autograd.grad(final.sum(), initial)[0], torch.ones_like(initial))
    _, final = ak.short_conv(x, weight, bias, "silu", return_final_state=True)
    assert not final.any()
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    empty, states = x[:1], torch.randn(3, 3, 16, device="cuda")
    assert torch.equal(ak.short_conv(empty, weight, bias, None, states, cu, True)[1], states)


def test_packing_out_of_range_is_cut_off():
    """Entries below zero, behind the tokens and descending: nothing is read or written out of range (the tensors lie inside
    larger ones whose surroundings stay as they were)."""
    c, total = 8, 40
    guard = torch.full((1, total + 64, c), 7.0, device="cuda")
    x = guard[:, 32:32 + total]
    weight, bias = torch.randn(c, 4, device="cuda"), torch.randn(c, device="cuda")
    for cu in ([0, 10, 1000, 2000], [5, -3, 20, 40], [0, 30, 10, 40], [-2 ** 31, 2 ** 31 - 1, 0, 2 ** 31 - 1]):
        out, final = ak.short_conv(x, weight, bias, "silu", None, torch.tensor(cu, dtype=torch.int32, device="cuda"), True)
        torch.cuda.synchronize()
        assert out.shape == x.shape and final.shape == (3, 3, c)
    assert (guard == 7.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c,w", [(1, 8, 4), (16, 1792, 4), (5, 131, 3), (9, 1025, 2), (300, 24, 4)])
def test_step(rows, c, w, dtype):
    x, weight, bias, initial = make(rows, 1, c, w, dtype)
    want, last = ak.short_conv(x, weight, bias, "silu", initial, return_final_state=True)
    state = initial.clone()
    out = ak.short_conv_step(x[:, 0], state, weight, bias, "silu")
    assert torch.equal(out, want[:, 0]) and torch.equal(state, last)
    check_forward(out[:, None], state, x, weight, bias, "silu", initial)


def test_step_slots():
    """Rows of padding, a cache whose slots lie apart, untouched slots, and a separate cache for the new states."""
    c, w, rows, pool = 72, 4, 7, 12
    x, weight, bias, _ = make(rows, 1, c, w, torch.bfloat16)
    larger = torch.randn(pool, 3, w - 1, c, device="cuda").to(torch.bfloat16)
    before = larger.clone()
    state = larger[:, 1]
    slots = torch.tensor([3, -1, 11, 0, 12, 5, -7], dtype=torch.int32, device="cuda")
    live = [0, 2, 3, 5]
    where = slots[live].long()
    want, last = ak.short_conv(x[live], weight, bias, None, state[where].contiguous(), return_final_state=True)
    apart = torch.full((pool, w - 1, c), 9.0, device="cuda", dtype=torch.bfloat16)
    out = ak.short_conv_step(x[:, 0], state, weight, bias, None, slots, apart)
    assert torch.equal(larger, before)
    expected = torch.full_like(apart, 9.0)
    expected[where] = last
    assert torch.equal(apart, expected)
    again = ak.short_conv_step(x[:, 0], state, weight, bias, None, slots)
    for o in (out, again):
        assert torch.equal(o[live], want[:, 0]) and not o[[1, 4, 6]].any()
    before[:, 1][where] = last
    assert torch.equal(larger, before)


@pytest.mark.parametrize("separate", [False, True])
def test_step_of_rows_that_share_a_slot(separate):
    c, w = 136, 4
    x, weight, bias, _ = make(6, 1, c, w, torch.float32)
    state = torch.randn(4, w - 1, c, device="cuda")
    slots = torch.tensor([2, 0, 2, 1, 2, 0], dtype=torch.int32, device="cuda")
    want, states = torch.empty(6, c, device="cuda"), state.clone()
    for r, s in enumerate(slots.tolist()):
        o, f = ak.short_conv(x[r:r + 1], weight, bias, "silu", states[s:s + 1].clone(), return_final_state=True)
        want[r], states[s] = o[0, 0], f[0]
    other = state.clone() if separate else None
    out = ak.short_conv_step(x[:, 0], state, weight, bias, "silu", slots, other)
    assert torch.equal(out, want) and torch.equal(other if separate else state, states)


def test_a_prompt_and_then_tokens_are_one_sequence():
    x, weight, bias, _ = make(2, 40, 64, 4, torch.float32)
    whole, end = ak.short_conv(x, weight, bias, "silu", return_final_state=True)
    first, state = ak.short_conv(x[:, :33], weight, bias, "silu", return_final_state=True)
    rest = [ak.short_conv_step(x[:, t], state, weight, bias, "silu") for t in range(33, 40)]
    assert torch.equal(torch.cat([first, torch.stack(rest, 1)], 1), whole) and torch.equal(state, end)


def test_repeats_bit_for_bit_and_on_a_stream_of_its_own():
    x, weight, bias, initial = make(3, 500, 264, 4, torch.bfloat16)

    def once():
        leaves = [t.detach().requires_grad_(True) for t in (x, weight, bias, initial)]
        out, final = ak.short_conv(*leaves[:3], "silu", leaves[3], return_final_state=True)
        return [out, final, *torch.autograd.grad([out, final], leaves, [torch.ones_like(out), torch.ones_like(final)])]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_captured_step_reads_the_slots_of_each_replay():
    c, w = 64, 4
    x, weight, bias, _ = make(4, 1, c, w, torch.float32)
    x = x[:, 0].contiguous()
    state, slots = torch.randn(8, w - 1, c, device="cuda"), torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    kept = state.clone()
    ak.short_conv_step(x, state, weight, bias, "silu", slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ak.short_conv_step(x, state, weight, bias, "silu", slots)
    for numbers in ([7, 3, -1, 5], [5, 5, 0, 1]):
        state.copy_(kept)
        slots.copy_(torch.tensor(numbers, dtype=torch.int32))
        x.copy_(torch.randn(4, c))
        graph.replay()
        torch.cuda.synchronize()
        eager = kept.clone()
        assert torch.equal(out, ak.short_conv_step(x, eager, weight, bias, "silu", slots)) and torch.equal(state, eager)


def test_gradients_cannot_be_differentiated_again():
    x, weight, bias, initial = make(1, 9, 8, 4, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, weight, bias, initial)]
    dout = torch.randn_like(x).requires_grad_(True)
    grads = torch.autograd.grad(ak.short_conv(*leaves[:3], "silu", leaves[3]), leaves, dout, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        grads[0].sum().backward()


def test_saved_tensors_that_change_are_an_error():
    x, weight, bias, initial = make(1, 9, 8, 4, torch.float32)
    weight.requires_grad_(True)
    out = ak.short_conv(x, weight, bias, "silu", initial)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), weight)
