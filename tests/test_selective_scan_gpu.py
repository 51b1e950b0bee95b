"""selective_scan and selective_scan_step against the recurrence in 64 bits, token by token.

Bounds.  Every value is a sum of products of inputs, decays and steps.  ``magnitudes`` runs the same formulas on the absolute
values of everything, which gives the sum of the magnitudes of all products that a value is made of.  A term that lived for
k tokens carries k roundings of the recurrence and k relative errors of the decay: each exp2 has 2 steps (4 half steps) and the
rounding of its argument, |dt A| half steps; softplus and the products add a fixed number (24, by its series and two
approximate instructions).  k is bounded by the length of the sequence, and the decays' arguments add up to what the term has
decayed by, which only shortens its life; so 6 L + 48 half steps of the magnitudes bound any value; sums over
channels and tokens (gradients of A, B, C, D, dt_bias) add one for each of their terms.

Decays and products below the smallest normal number, 2^-126, are taken as zero (the exponential flushes them).  A term that
is lost that way is 2^-126 of what it decayed from, a product of at most three inputs that are drawn from a normal
distribution (none of them reaches 6.4, so 2^8 bounds it); with L terms in a value that is L 2^-118."""
import pytest
import torch

import ascend_kernel as ak
from operator_checks import differences, near, scan_plain

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(b, l, c, n, g, dtype, full=True, start=True, sliced=False, states=None, seed=None):
    if seed is not None:
        torch.manual_seed(seed)

    def act(*inner, scale=1.0):
        size = torch.Size(inner).numel()
        if sliced:  # column slices of a wider matrix, at an odd place
            wide = (torch.randn(b, l, size + 10, device="cuda") * scale).to(dtype)
            return wide[..., 5:5 + size].unflatten(-1, inner)
        return (torch.randn(b, l, *inner, device="cuda") * scale).to(dtype)

    x, dt = act(c), act(c, scale=0.7)
    A = -(torch.arange(1, n + 1, device="cuda") * torch.exp(0.2 * torch.randn(c, n, device="cuda")))
    B, C = act(g, n), act(g, n)
    D = torch.randn(c, device="cuda") if full else None
    z = act(c) if full else None
    bias = torch.randn(c, device="cuda") - 2.0 if full else None
    initial = torch.randn(states or b, c, n, device="cuda") if start else None
    return x, dt, A, B, C, D, z, bias, initial


def double(t):
    return None if t is None else t.detach().double()


def magnitudes(x, dt, A, B, C, D, z, bias, softplus, start):
    """The forward call on absolute values (decays as they are)."""
    step = dt.double() if bias is None else dt.double() + bias.double()
    if softplus:
        step = torch.logaddexp(step, torch.zeros_like(step))
    out, h = scan_plain(x.double().abs(), step, A.double(), B.double().abs(), C.double().abs(),
                        None if D is None else D.double().abs(), None, None, False, None if start is None else start.double().abs())
    return (out if z is None else out * z.double().abs()), h


def rounding_count(l):
    return 6 * l + 48


def flush(l):
    return l * 2.0 ** -118


CASES = [
    # b, l, c, n, g, full, start, sliced
    (1, 1, 1, 1, 1, True, True, False), (1, 1, 64, 16, 1, True, False, False), (2, 3, 34, 4, 1, True, True, False),
    (1, 33, 96, 16, 1, False, True, False), (3, 64, 65, 16, 1, True, True, False), (2, 131, 130, 16, 2, True, True, True),
    (1, 257, 128, 24, 4, True, True, False), (2, 100, 66, 64, 1, True, False, False), (1, 70, 40, 128, 1, True, True, False),
    (1, 90, 36, 7, 3, True, True, False), (1, 700, 192, 16, 1, True, True, False), (2, 450, 100, 33, 1, False, False, True),
    (1, 1200, 8, 16, 1, True, True, False),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,l,c,n,g,full,start,sliced", CASES)
def test_forward(b, l, c, n, g, full, start, sliced, dtype):
    x, dt, A, B, C, D, z, bias, initial = make(b, l, c, n, g, dtype, full, start, sliced)
    softplus = full
    if not softplus:
        dt = dt.abs() * 0.1
    out, final = ak.selective_scan(x, dt, A, B, C, D, z, bias, softplus, initial, return_final_state=True)
    want, last = scan_plain(*map(double, (x, dt, A, B, C, D, z, bias)), softplus, double(initial))
    top, top_h = magnitudes(x, dt, A, B, C, D, z, bias, softplus, initial)
    assert out.dtype is dtype and out.is_contiguous() and final.dtype is torch.float32
    near(out, want, top, rounding_count(l), "out", flush(l))
    near(final, last, top_h, rounding_count(l), "final", flush(l))
    assert torch.equal(out, ak.selective_scan(x, dt, A, B, C, D, z, bias, softplus, initial))


def plain_gradients(tensors, softplus, dout, dfinal):
    """Gradients in 64 bits, and the magnitudes of what they are made of: the same gradients on absolute values (every factor
    of every product in the formulas is taken without its sign; the derivatives of the activations are below 1.1)."""
    x, dt, A, B, C, D, z, bias, initial = tensors
    leaves = [t.detach().double().requires_grad_(True) for t in tensors if t is not None]
    it = iter(leaves)
    full = [None if t is None else next(it) for t in tensors]
    out, final = scan_plain(*full[:8], softplus, full[8])
    grads = iter(torch.autograd.grad([out, final], leaves, [dout.double(), dfinal.double()]))
    grads = [None if t is None else next(grads) for t in tensors]
    with torch.no_grad():
        step = double(dt) if bias is None else double(dt) + double(bias)
        if softplus:
            step = torch.logaddexp(step, torch.zeros_like(step))
        step = step.abs()
        per = x.shape[2] // B.shape[2]
        Bm, Cm = (t.double().abs().repeat_interleave(per, 2) for t in (B, C))
        xm, Am = x.double().abs(), A.double().abs()
        zm = 1 if z is None else z.double().abs()
        dy = dout.double().abs() * zm
        skip = 0 if D is None else D.double().abs()
        h = torch.zeros(x.shape[0], *A.shape, dtype=torch.float64, device="cuda") if initial is None else initial.double().abs()
        states = [h]
        for t in range(x.shape[1]):
            h = torch.exp(step[:, t, :, None] * A.double()) * h + (step[:, t] * xm[:, t])[..., None] * Bm[:, t]
            states.append(h)
        g = dfinal.double().abs()
        top = {k: [] for k in ("x", "dt", "B", "C", "y")}
        top_a = torch.zeros_like(Am)
        for t in reversed(range(x.shape[1])):
            g = g + dy[:, t, :, None] * Cm[:, t]
            groups = (x.shape[0], B.shape[2], per, A.shape[1])
            top["C"].append((states[t + 1] * dy[:, t, :, None]).view(groups).sum(2))
            top["B"].append((g * (step[:, t] * xm[:, t])[..., None]).view(groups).sum(2))
            through = (g * Bm[:, t]).sum(-1)
            g = g * torch.exp(step[:, t, :, None] * A.double())
            q = g * states[t]
            top["x"].append(step[:, t] * through + dy[:, t] * skip)
            top["dt"].append(xm[:, t] * through + (q * Am).sum(-1))
            top["y"].append((states[t + 1] * Cm[:, t]).sum(-1) + skip * xm[:, t])
            top_a += (q * step[:, t, :, None]).sum(0)
        top = {k: torch.stack(v[::-1], 1) for k, v in top.items()}
        magnitude = [top["x"], top["dt"], top_a, top["B"], top["C"], (dy * xm).sum((0, 1)),
                     1.1 * dout.double().abs() * top["y"], top["dt"].sum((0, 1)), g]
    return grads, magnitude


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,l,c,n,g,full,start,sliced", CASES)
def test_gradients(b, l, c, n, g, full, start, sliced, dtype):
    tensors = list(make(b, l, c, n, g, dtype, full, start, sliced))
    if not full:
        tensors[1] = tensors[1].abs() * 0.1
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in tensors]
    x, dt, A, B, C, D, z, bias, initial = leaves
    out, final = ak.selective_scan(x, dt, A, B, C, D, z, bias, full, initial, return_final_state=True)
    dout, dfinal = torch.randn_like(out), torch.randn_like(final)
    got = iter(torch.autograd.grad([out, final], [t for t in leaves if t is not None], [dout, dfinal]))
    got = [None if t is None else next(got) for t in leaves]
    want, tops = plain_gradients([None if t is None else t.detach() for t in leaves], full, dout, dfinal)
    ops = 2 * rounding_count(l) + 16
    many = {2: b * l, 3: c, 4: c, 5: b * l, 7: b * l}
    for i, name in enumerate(("dx", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dinitial")):
        if got[i] is not None:
            assert got[i].dtype is leaves[i].dtype
            near(got[i], want[i], tops[i], ops + many.get(i, 0), name, flush(l))


def test_against_differences():
    tensors = make(1, 21, 6, 5, 2, torch.float32, seed=5)
    coefficients = torch.randn(1, 21, 6, device="cuda"), torch.randn(1, 6, 5, device="cuda")

    def f(*leaves):
        out, final = ak.selective_scan(*leaves[:8], True, leaves[8], return_final_state=True)
        parts = torch.cat([(out * coefficients[0]).flatten(), (final * coefficients[1]).flatten()]).double()
        return parts.sum(), parts.abs().sum()

    leaves = [t.requires_grad_(True) for t in tensors]
    out, final = ak.selective_scan(*leaves[:8], True, leaves[8], return_final_state=True)
    differences(f, leaves, torch.autograd.grad([out, final], leaves, list(coefficients)), 6)


def test_each_gradient_alone_and_missing_upstream():
    tensors = make(2, 70, 40, 16, 1, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in tensors]
    out, final = ak.selective_scan(*leaves[:8], True, leaves[8], return_final_state=True)
    dout, dfinal = torch.randn_like(out), torch.randn_like(final)
    every = torch.autograd.grad([out, final], leaves, [dout, dfinal], retain_graph=True)
    for i in range(9):
        alone = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        o, f = ak.selective_scan(*alone[:8], True, alone[8], return_final_state=True)
        assert torch.equal(torch.autograd.grad([o, f], alone[i], [dout, dfinal])[0], every[i])
    from_out = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    zeros = torch.autograd.grad([out, final], leaves, [dout, torch.zeros_like(final)], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(from_out, zeros))
    from_final = torch.autograd.grad(final, leaves, dfinal, retain_graph=True, allow_unused=True)
    zeros = torch.autograd.grad([out, final], leaves, [torch.zeros_like(out), dfinal], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(from_final, zeros))
    broadcast = torch.autograd.grad(out.sum(), leaves[0])[0]
    assert broadcast.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths,behind,c,n", [([5], 0, 16, 16), ([1, 0, 2, 37, 0, 130, 3, 0], 5, 72, 16), ([0, 0], 3, 9, 8),
                                                ([300, 1, 64, 1, 199, 65], 0, 34, 16), ([2] * 260, 70, 8, 4)])
def test_packed_sequences(lengths, behind, c, n, dtype):
    total, count = sum(lengths) + behind, len(lengths)
    tensors = make(1, total, c, n, 1, dtype, sliced=True, states=count)
    cu = torch.tensor([0] + lengths).cumsum(0).to("cuda", torch.int32)
    leaves = [t.detach().requires_grad_(True) for t in tensors]
    out, final = ak.selective_scan(*leaves[:8], True, leaves[8], cu, True)
    dout, dfinal = torch.randn_like(out), torch.randn_like(final)
    grads = torch.autograd.grad([out, final], leaves, [dout, dfinal])
    with torch.no_grad():
        again = ak.selective_scan(*tensors[:8], True, tensors[8], cu, True)
    assert torch.equal(again[0], out) and torch.equal(again[1], final)
    at, da, da_top = 0, 0, 0
    longest = max(lengths)
    seen = set()
    for s, m in enumerate(lengths):
        own = slice(at, at + m)
        at += m
        if m == 0:
            assert torch.equal(final[s], tensors[8][s]) and torch.equal(grads[8][s], dfinal[s])
            continue
        if len(lengths) > 20 and s % 13:  # many alike: some of them
            continue
        x, dt, A, B, C, D, z, bias, initial = [t[:, own] if t.dim() > 2 and t.shape[1] == total and i not in (2, 8) else t
                                               for i, t in enumerate(tensors)]
        part = [x, dt, A, B, C, D, z, bias, initial[s:s + 1]]
        want, last = scan_plain(*map(double, part[:8]), True, double(part[8]))
        top, top_h = magnitudes(*part[:8], True, part[8])
        near(out.detach()[:, own], want, top, rounding_count(m), f"out {s}", flush(m))
        near(final.detach()[s:s + 1], last, top_h, rounding_count(m), f"final {s}", flush(m))
        expected, tops = plain_gradients(part, True, dout[:, own], dfinal[s:s + 1])
        for i in (0, 1, 3, 4, 6):
            near(grads[i][:, own], expected[i], tops[i], 2 * rounding_count(m) + 16 + c, f"gradient {i} of {s}", flush(m))
        near(grads[8][s:s + 1], expected[8], tops[8], 2 * rounding_count(m) + 16, f"dinitial {s}", flush(m))
        da, da_top = da + expected[2], da_top + tops[2]
        seen.add(s)
    if len(lengths) <= 20:
        near(grads[2], da if torch.is_tensor(da) else torch.zeros_like(grads[2]).double(),
             da_top if torch.is_tensor(da_top) else torch.zeros_like(grads[2]).double(),
             2 * rounding_count(longest) + 16 + total, "dA", flush(total))
    for i in (0, 1, 3, 4, 6):
        assert not grads[i][:, at:].any()
    assert not out[:, at:].any()


def test_no_tokens():
    x, dt, A, B, C, D, z, bias, initial = make(2, 0, 16, 4, 1, torch.float32)
    out, final = ak.selective_scan(x, dt, A, B, C, D, z, bias, True, initial, return_final_state=True)
    assert out.shape == (2, 0, 16) and torch.equal(final, initial)
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    states = torch.randn(3, 16, 4, device="cuda", requires_grad=True)
    _, final = ak.selective_scan(*(t[:1] if i in (0, 1, 3, 4, 6) else t for i, t in enumerate((x, dt, A, B, C, D, z, bias))), True,
                                 states, cu, True)
    assert torch.equal(final, states)
    assert torch.equal(torch.autograd.grad(final, states, 2 * torch.ones_like(final))[0], torch.full_like(states, 2.0))


def test_packing_out_of_range_is_cut_off():
    c, n, total = 40, 16, 200
    tensors = make(1, total, c, n, 1, torch.float32, start=False)
    for cu in ([0, 10, 1000, 2000], [5, -3, 20, 200], [0, 130, 10, 200], [-2 ** 31, 2 ** 31 - 1, 0, 2 ** 31 - 1]):
        leaves = [t.detach().requires_grad_(True) for t in tensors[:8]]
        cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
        out, final = ak.selective_scan(*leaves, True, None, cu, True)
        torch.autograd.grad([out.sum(), final.sum()], leaves)
        torch.cuda.synchronize()
        assert out.shape == tensors[0].shape and final.shape == (3, c, n)


def test_segments_do_not_change_the_result():
    """A long sequence of few channels is cut into segments; many rows of the same channels are not."""
    tensors = make(1, 3000, 64, 16, 1, torch.float32, seed=8)
    rows = 80
    out, final = ak.selective_scan(*tensors[:8], True, tensors[8], return_final_state=True)
    many = [t.expand(rows, *t.shape[1:]).contiguous() if i in (0, 1, 3, 4, 6, 8) else t for i, t in enumerate(tensors)]
    wide, last = ak.selective_scan(*many[:8], True, many[8], return_final_state=True)
    top, top_h = magnitudes(*tensors[:8], True, tensors[8])
    near(out, wide[:1].double(), top, rounding_count(3000))
    near(final, last[:1].double(), top_h, rounding_count(3000))
    assert all(torch.equal(wide[0], wide[r]) for r in range(1, rows))


def test_extreme_steps():
    """softplus at both ends: steps that vanish keep the state, and steps that are large forget it."""
    c, n = 32, 16
    tensors = make(1, 12, c, n, 1, torch.float32)
    for raw, forget in ((-200.0, False), (-30.0, False), (60.0, True), (300.0, True)):
        x, dt, A, B, C, D, z, bias, initial = tensors
        dt = torch.full_like(dt, raw)
        out, final = ak.selective_scan(x, dt, A, B, C, D, z, None, True, initial, return_final_state=True)
        want, last = scan_plain(*map(double, (x, dt, A, B, C, D, z, None)), True, double(initial))
        top, top_h = magnitudes(x, dt, A, B, C, D, z, None, True, initial)
        near(out, want, top, rounding_count(12), flushed=flush(12))
        near(final, last, top_h, rounding_count(12), flushed=flush(12))


def step_inputs(tensors):
    x, dt, A, B, C, D, z, bias, _ = tensors
    return (x[:, 0], dt[:, 0], A, B[:, 0], C[:, 0]), dict(D=D, z=None if z is None else z[:, 0], dt_bias=bias, dt_softplus=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c,n,g,full", [(1, 8, 16, 1, True), (16, 1536, 16, 1, True), (5, 131, 7, 1, True), (9, 66, 64, 2, True),
                                             (70, 260, 128, 1, False), (300, 48, 24, 4, True), (130, 1024, 16, 1, True)])
@pytest.mark.parametrize("sliced", [False, True])
def test_step(rows, c, n, g, full, sliced, dtype):
    tensors = make(rows, 1, c, n, g, dtype, full, True, sliced)
    arguments, options = step_inputs(tensors)
    state = tensors[8].clone()
    out = ak.selective_scan_step(*arguments, state, **options)
    x, dt, A, B, C, D, z, bias, initial = tensors
    want, last = scan_plain(*map(double, (x, dt, A, B, C, D, z, bias)), True, double(initial))
    top, top_h = magnitudes(x, dt, A, B, C, D, z, bias, True, initial)
    near(out, want[:, 0], top[:, 0], rounding_count(1), flushed=flush(1))
    near(state, last, top_h, rounding_count(1), flushed=flush(1))


@pytest.mark.parametrize("rows", [7, 700])
def test_step_slots(rows):
    c, n = 72, 16
    pool = rows + 30
    tensors = make(rows, 1, c, n, 1, torch.bfloat16, start=False)
    arguments, options = step_inputs(tensors)
    larger = torch.randn(pool, 3, c, n, device="cuda")
    before, state = larger.clone(), larger[:, 1]
    slots = torch.randperm(pool)[:rows].to(torch.int32)
    slots[1], slots[rows - 1], slots[rows - 3] = -1, pool, -2 ** 31
    dead = [1, rows - 3, rows - 1]
    live = [r for r in range(rows) if r not in dead]
    slots = slots.cuda()
    where = slots[live].long()
    own = state[where].contiguous()
    picked = [t[live] if i != 2 else t for i, t in enumerate(arguments)]
    want = ak.selective_scan_step(*picked, own, **{**options, "z": options["z"][live]})
    apart = torch.full((pool, c, n), 9.0, device="cuda")
    out = ak.selective_scan_step(*arguments, state, **options, slots=slots, state_out=apart)
    assert torch.equal(larger, before)
    expected = torch.full_like(apart, 9.0)
    expected[where] = own
    assert torch.equal(apart, expected)
    again = ak.selective_scan_step(*arguments, state, **options, slots=slots)
    for o in (out, again):
        assert torch.equal(o[live], want) and not o[dead].any()
    before[:, 1][where] = own
    assert torch.equal(larger, before)


@pytest.mark.parametrize("rows", [6, 900])
@pytest.mark.parametrize("separate", [False, True])
def test_step_of_rows_that_share_a_slot(rows, separate):
    c, n, pool = 48, 16, 5
    tensors = make(rows, 1, c, n, 1, torch.float32, start=False)
    arguments, options = step_inputs(tensors)
    state = torch.randn(pool, c, n, device="cuda")
    slots = torch.randint(0, pool, (rows,)).to(torch.int32)
    want, states = torch.empty(rows, c, device="cuda"), state.clone()
    for r, s in enumerate(slots.tolist()):
        one = [t[r:r + 1] if i != 2 else t for i, t in enumerate(arguments)]
        want[r] = ak.selective_scan_step(*one, states[s:s + 1], **{**options, "z": options["z"][r:r + 1]})[0]
    other = state.clone() if separate else None
    out = ak.selective_scan_step(*arguments, state, **options, slots=slots.cuda(), state_out=other)
    assert torch.equal(out, want) and torch.equal(other if separate else state, states)


def test_repeats_bit_for_bit_and_on_a_stream_of_its_own():
    tensors = make(2, 500, 200, 16, 1, torch.bfloat16)

    def once():
        leaves = [t.detach().requires_grad_(True) for t in tensors]
        out, final = ak.selective_scan(*leaves[:8], True, leaves[8], return_final_state=True)
        return [out, final, *torch.autograd.grad([out, final], leaves, [torch.ones_like(out), torch.ones_like(final)])]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_captured_training_step_and_generation_step():
    tensors = make(2, 300, 64, 16, 1, torch.bfloat16)
    step_tensors = make(4, 1, 64, 16, 1, torch.bfloat16, start=False)
    arguments, options = step_inputs(step_tensors)
    state, slots = torch.randn(8, 64, 16, device="cuda"), torch.tensor([0, 5, 2, 7], dtype=torch.int32, device="cuda")
    other = torch.zeros_like(state)

    def once():
        leaves = [t.detach().requires_grad_(True) for t in tensors]
        out, final = ak.selective_scan(*leaves[:8], True, leaves[8], return_final_state=True)
        grads = torch.autograd.grad([out, final], leaves, [tensors[0], tensors[8]])
        return [out.detach(), final.detach(), *grads,
                ak.selective_scan_step(*arguments, state, **options, slots=slots, state_out=other)]

    once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = once()
    tensors[0].copy_(torch.randn_like(tensors[0]))
    slots.copy_(torch.tensor([1, 1, -1, 3], dtype=torch.int32))
    other.zero_()
    graph.replay()
    torch.cuda.synchronize()
    kept = other.clone()
    other.zero_()
    eager = once()
    assert all(torch.equal(a, b) for a, b in zip(captured, eager)) and torch.equal(kept, other)


def test_a_prompt_and_then_tokens_are_one_sequence():
    tensors = make(2, 40, 64, 16, 1, torch.float32)
    x, dt, A, B, C, D, z, bias, initial = tensors
    whole, end = ak.selective_scan(x, dt, A, B, C, D, z, bias, True, initial, return_final_state=True)
    cut = [t[:, :33] if i in (0, 1, 3, 4, 6) else t for i, t in enumerate(tensors)]
    first, state = ak.selective_scan(*cut[:8], True, cut[8], return_final_state=True)
    rest = []
    for t in range(33, 40):
        one = [v[:, t:t + 1] if i in (0, 1, 3, 4, 6) else v for i, v in enumerate(tensors)]
        arguments, options = step_inputs(one)
        rest.append(ak.selective_scan_step(*arguments, state, **options))
    top, top_h = magnitudes(*tensors[:8], True, initial)
    near(torch.cat([first, torch.stack(rest, 1)], 1), whole.double(), top, rounding_count(40))
    near(state, end.double(), top_h, rounding_count(40))


def test_columns_that_keep_nothing():
    """A = -inf: such a column is the last token's own contribution; lengths that end inside a tile, and inside a chunk."""
    for l in (5, 33, 70):
        x, dt, A, B, C, D, z, bias, initial = make(1, l, 40, 16, 1, torch.float32)
        A[::3, 2] = float("-inf")
        A[1] = float("-inf")
        leaves = [t.detach().requires_grad_(True) for t in (x, dt, A, B, C, D, z, bias, initial)]
        out, final = ak.selective_scan(*leaves[:8], True, leaves[8], return_final_state=True)
        want, last = scan_plain(*map(double, (x, dt, A, B, C, D, z, bias)), True, double(initial))
        top, top_h = magnitudes(x, dt, A, B, C, D, z, bias, True, initial)
        near(out.detach(), want, top, rounding_count(l), flushed=flush(l))
        near(final.detach(), last, top_h, rounding_count(l), flushed=flush(l))
        for g in torch.autograd.grad([out, final], leaves, [torch.ones_like(out), torch.ones_like(final)]):
            assert g.isfinite().all()
        state = initial.clone()
        arguments, options = step_inputs([t[:, :1] if i in (0, 1, 3, 4, 6) else t for i, t in enumerate(
            (x, dt, A, B, C, D, z, bias, initial))])
        ak.selective_scan_step(*arguments, state, **options)
        assert state.isfinite().all()


def test_what_lies_behind_or_in_other_sequences_does_not_spread():
    """Infinities and NaN behind the last packed sequence, in a neighbouring sequence and in rows of padding."""
    lengths, c, n = [20, 45, 30], 36, 16
    total = sum(lengths) + 9
    tensors = make(1, total, c, n, 1, torch.float32, states=3)
    cu = torch.tensor([0] + lengths).cumsum(0).to("cuda", torch.int32)
    spoilt = [t.clone() for t in tensors]
    for i in (0, 1, 3, 4, 6):
        spoilt[i][:, sum(lengths):] = float("nan")
        spoilt[i][:, 20:65] = float("inf")
    results = []
    for ts in (tensors, spoilt):
        leaves = [t.detach().requires_grad_(True) for t in ts]
        out, final = ak.selective_scan(*leaves[:8], True, leaves[8], cu, True)
        dout = torch.ones_like(out)
        dout[:, sum(lengths):] = float("nan")
        grads = torch.autograd.grad([out, final], [leaves[i] for i in (0, 1, 3, 4, 6)], [dout, torch.ones_like(final)])
        results.append([out.detach(), *grads])
        states = final.detach()[[0, 2]]
        results[-1].append(states)
    for good, bad in zip(*results):
        if good.shape[1] == total:
            for own in (slice(0, 20), slice(65, 95), slice(95, total)):
                assert torch.equal(good[:, own], bad[:, own])
        else:
            assert torch.equal(good, bad)
    step = make(4, 1, c, n, 1, torch.float32, start=False)
    step[0][2] = float("nan")
    arguments, options = step_inputs(step)
    state = torch.randn(6, c, n, device="cuda")
    state[5] = float("nan")
    out = ak.selective_scan_step(*arguments, state, **options, slots=torch.tensor([1, 0, -1, 3], dtype=torch.int32, device="cuda"))
    assert out.isfinite().all() and not out[2].any() and state[:5].isfinite().all() and state[5].isnan().all()


def test_offsets_past_32_bits():
    """More than 2^31 elements in the activations, and in a cache of states; what lies at their end equals the same alone."""
    c, n, tail = 4096, 4, 96
    total = 2 ** 31 // c + 1000
    x = torch.zeros(1, total, c, device="cuda", dtype=torch.bfloat16)
    B, C = (torch.randn(1, total, 1, n, device="cuda").to(torch.bfloat16) for _ in range(2))
    x[:, -tail:] = torch.randn(1, tail, c, device="cuda").to(torch.bfloat16)
    A = -torch.rand(c, n, device="cuda")
    cu = torch.tensor([0, total - tail, total], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        out, final = ak.selective_scan(x, x, A, B, C, dt_softplus=True, cu_seqlens=cu, return_final_state=True)
        end = [t[:, -tail:].contiguous() for t in (x, B, C)]
        want, last = ak.selective_scan(end[0], end[0], A, end[1], end[2], dt_softplus=True, return_final_state=True)
        top, top_h = magnitudes(end[0], end[0], A, end[1], end[2], None, None, None, True, None)
        near(out[:, -tail:], want.double(), top, 2 * rounding_count(tail))
        near(final[1:], last.double(), top_h, 2 * rounding_count(tail))
        assert not out[:, :-tail].any()
        del out
        weight = torch.randn(c, 4, device="cuda")
        conv, held = ak.short_conv(x, weight, None, "silu", None, cu, True)
        alone, ends = ak.short_conv(end[0], weight, None, "silu", return_final_state=True)
        assert torch.equal(conv[:, -tail:], alone) and torch.equal(held[1:], ends)
        del conv
        # how a row's squares are added up depends on the number of rows: a value may fall on the other side of a border
        # between two numbers of the type, one step away (2^-7 of it in bf16, 2^-3 in e4m3)
        ones = torch.ones(c, device="cuda")
        for f, step in ((lambda t: ak.rms_norm(t, ones), 2.0 ** -7), (lambda t: ak.rms_norm_quant(t, ones)[0], 2.0 ** -3)):
            there, here = f(x)[:, -tail:].float(), f(end[0]).float()
            assert ((there - here).abs() <= step * torch.maximum(there.abs(), here.abs())).all() and here.any(-1).all()
        del x
        wide = 128
        slots = 2 ** 31 // (c * wide) + 3
        cache = torch.empty(slots, c, wide, device="cuda")
        cache[-1] = torch.randn(c, wide, device="cuda")
        state = cache[-1:].clone()
        tensors = make(1, 1, c, wide, 1, torch.float32, start=False)
        arguments, options = step_inputs(tensors)
        one = ak.selective_scan_step(*arguments, cache, **options, slots=torch.tensor([slots - 1], dtype=torch.int32, device="cuda"))
        assert torch.equal(one, ak.selective_scan_step(*arguments, state, **options)) and torch.equal(cache[-1:], state)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,l,c,n,g,gated,skip", [
    (1, 256, 64, 8, 1, True, True), (9, 257, 512, 8, 1, False, True), (2, 300, 64, 16, 2, True, False),
    (9, 289, 512, 16, 1, False, False), (1, 290, 68, 32, 1, True, True), (1, 260, 36, 64, 1, True, True),
    (1, 256, 32, 128, 1, True, False), (3, 273, 40, 12, 1, True, True),
])
def test_forward_of_long_sequences(b, l, c, n, g, gated, skip, dtype):
    x, dt, A, B, C, D, z, bias, initial = make(b, l, c, n, g, dtype, seed=3)
    D, z = D if skip else None, z if gated else None
    out, final = ak.selective_scan(x, dt, A, B, C, D, z, bias, True, initial, return_final_state=True)
    want, last = scan_plain(*map(double, (x, dt, A, B, C, D, z, bias)), True, double(initial))
    top, top_h = magnitudes(x, dt, A, B, C, D, z, bias, True, initial)
    near(out, want, top, rounding_count(l), "out", flush(l))
    near(final, last, top_h, rounding_count(l), "final", flush(l))


@pytest.mark.parametrize("dtype", DTYPES)
def test_forward_of_long_packed_sequences(dtype):
    lengths = [700, 0, 1, 33, 0, 1025, 290]
    l, c, n = sum(lengths) + 7, 72, 16  # seven tokens behind the last sequence
    x, dt, A, B, C, D, z, bias, initial = make(1, l, c, n, 2, dtype, states=len(lengths), seed=4)
    edges = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    out, final = ak.selective_scan(x, dt, A, B, C, D, z, bias, True, initial, cu_seqlens=edges, return_final_state=True)
    assert not out[:, l - 7:].any()
    at = 0
    for i, m in enumerate(lengths):
        if m == 0:
            assert torch.equal(final[i], initial[i])
            continue
        part = [None if t is None else t[:, at:at + m] for t in (x, dt, B, C, z)]
        args = part[0], part[1], A, part[2], part[3], D, part[4], bias
        want, last = scan_plain(*map(double, args), True, double(initial[i:i + 1]))
        top, top_h = magnitudes(*args, True, initial[i:i + 1])
        near(out[:, at:at + m], want, top, rounding_count(m), f"out {i}", flush(m))
        near(final[i:i + 1], last, top_h, rounding_count(m), f"final {i}", flush(m))
        at += m


def test_long_segments_against_two_calls():
    """A sequence of a few channels is cut into segments; the same one as two calls, joined by their states, is cut elsewhere.

    All inputs are positive and dt is at least 0.05 with A at most -1, so that a term is below 2^-24 of its start after 340 tokens,
    which bounds its roundings as at the top: 6 * 340 + 48 half steps of the value itself and one half step for what is behind, on
    both sides.  Gradients of B and C add 64 channels, those of A the sums of 64 tokens and their joint sums."""
    torch.manual_seed(5)
    l, c, n = 40064, 64, 16
    x, B, C, dout = (torch.rand(1, l, w, device="cuda") + 0.1 for w in (c, n, n, c))
    dt = torch.rand(1, l, c, device="cuda") * 0.1 + 0.05
    A = -(torch.rand(c, n, device="cuda") + 1)
    start, dfinal = torch.rand(1, c, n, device="cuda"), torch.rand(1, c, n, device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, A, B, C, start)]
    x, A, B, C, start = leaves

    def call(a, b, state):
        return ak.selective_scan(x[:, a:b], dt[:, a:b], A, B[:, a:b, None], C[:, a:b, None], initial_states=state,
                                 return_final_state=True)

    out, final = call(0, l, start)
    got = [out, final, *torch.autograd.grad([out, final], leaves, [dout, dfinal])]
    half = 12000
    first, state = call(0, half, start)
    second, last = call(half, l, state)
    both = torch.cat([first, second], 1)
    want = [both, last, *torch.autograd.grad([both, last], leaves, [dout, dfinal])]
    life = 6 * 340 + 50
    for name, a, b, count in zip(("out", "final", "dx", "dA", "dB", "dC", "dinitial"), got, want,
                                 (life, life, life, life + 64 + l // 64, life + 64, life + 64, life)):
        near(a, b.double(), b.double().abs(), 2 * count, name, flush(l))
