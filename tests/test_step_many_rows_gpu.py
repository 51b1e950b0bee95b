"""The kernels of the generation steps that take four rows of the batch at a time, which full batches reach: every state size and
layout, a last CTA with fewer rows, rows of padding, and slots that rows share within a CTA and across them.

Bounds are those of test_selective_scan_gpu.py and test_short_conv_gpu.py."""
import pytest
import torch

import ascend_kernel as ak
from operator_checks import near, scan_plain
from test_selective_scan_gpu import double, flush, magnitudes, make, rounding_count, step_inputs
from test_short_conv_gpu import check_forward
from test_short_conv_gpu import make as make_conv

pytestmark = pytest.mark.gpu

F32, BF16, F16 = DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def channels_of_a_cta(n):
    lanes = 1
    while 8 * lanes < n:
        lanes *= 2
    return 128 // lanes


def shared_slots(rows, pool):
    """Numbers of slots: most are shared, some by neighbouring rows of one CTA; rows of padding between."""
    slots = torch.randint(0, pool, (rows,))
    slots[4:8] = torch.tensor([2, 2, -1, 2])
    slots[rows - 3:] = torch.tensor([pool, 2, 1])
    slots[::29] = -1
    return slots.to(torch.int32)


SCAN_ROWS = [(2403, 72, 16, 1), (2401, 131, 8, 1), (2402, 40, 32, 2), (1203, 66, 64, 1), (1201, 34, 128, 1), (2401, 72, 7, 1), (2403, 50, 33, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c,n,g", SCAN_ROWS)
def test_scan_step_of_many_rows(rows, c, n, g, dtype):
    blocks = g * -(-(c // g) // channels_of_a_cta(n))
    assert rows * blocks >= 16 * sms() and rows % 4
    tensors = make(rows, 1, c, n, g, dtype, seed=rows)
    arguments, options = step_inputs(tensors)
    x, dt, A, B, C, D, z, bias, initial = tensors
    state = initial.clone()
    out = ak.selective_scan_step(*arguments, state, **options)
    want, last = scan_plain(*map(double, (x, dt, A, B, C, D, z, bias)), True, double(initial))
    top, top_h = magnitudes(x, dt, A, B, C, D, z, bias, True, initial)
    near(out, want[:, 0], top[:, 0], rounding_count(1), flushed=flush(1))
    near(state, last, top_h, rounding_count(1), flushed=flush(1))


@pytest.mark.parametrize("dtype,odd", [(F32, False), (BF16, False), (F16, True)])
@pytest.mark.parametrize("rows,c,n,g", SCAN_ROWS[:1] + SCAN_ROWS[2:4])
@pytest.mark.parametrize("separate", [False, True])
def test_scan_step_of_many_rows_that_share_slots(rows, c, n, g, dtype, odd, separate):
    """Against one row at a time; slots at an odd place (single loads) and aligned."""
    pool = 300
    arguments, options = step_inputs(make(rows, 1, c, n, g, dtype, start=False, seed=rows))
    whole = torch.randn(pool, c * n + (5 if odd else 8), device="cuda")
    state = whole[:, (3 if odd else 8):][:, :c * n].unflatten(-1, (c, n))
    kept, slots = whole.clone(), shared_slots(rows, pool)
    own = state.clone()
    want = torch.zeros(rows, c, device="cuda", dtype=dtype)
    for r, s in enumerate(slots.tolist()):
        if 0 <= s < pool:
            one = [t[r:r + 1] if i != 2 else t for i, t in enumerate(arguments)]
            want[r] = ak.selective_scan_step(*one, own[s:s + 1], **{**options, "z": options["z"][r:r + 1]})[0]
    other = state.contiguous() if separate else None
    out = ak.selective_scan_step(*arguments, state, **options, slots=slots.cuda(), state_out=other)
    assert torch.equal(out, want) and torch.equal(other if separate else state, own)
    if separate:
        assert torch.equal(whole, kept)
    else:
        assert torch.equal(whole[:, :3], kept[:, :3])


CONV_ROWS = [(1203, 136, 4), (1201, 131, 3), (1206, 64, 2), (605, 520, 4)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c,w", CONV_ROWS)
def test_convolution_step_of_many_rows(rows, c, w, dtype):
    assert rows * -(-c // 512) >= 8 * sms() and rows % 4
    x, weight, bias, initial = make_conv(rows, 1, c, w, dtype)
    want, last = ak.short_conv(x, weight, bias, "silu", initial, return_final_state=True)
    state = initial.clone()
    out = ak.short_conv_step(x[:, 0], state, weight, bias, "silu")
    assert torch.equal(out, want[:, 0]) and torch.equal(state, last)
    check_forward(out[:, None], state, x, weight, bias, "silu", initial)


@pytest.mark.parametrize("dtype,odd", [(F32, False), (BF16, False), (F16, True)])
@pytest.mark.parametrize("rows,c,w", CONV_ROWS)
@pytest.mark.parametrize("separate", [False, True])
def test_convolution_step_of_many_rows_that_share_slots(rows, c, w, dtype, odd, separate):
    pool, held = 300, w - 1
    x, weight, bias, _ = make_conv(rows, 1, c, w, dtype, start=False)
    x = x[:, 0]
    whole = torch.randn(pool, held * c + (5 if odd else 8), device="cuda").to(dtype)
    state = whole[:, (3 if odd else 8):][:, :held * c].unflatten(-1, (held, c))
    kept, slots = whole.clone(), shared_slots(rows, pool)
    own, want = state.clone(), torch.zeros(rows, c, device="cuda", dtype=dtype)
    for r, s in enumerate(slots.tolist()):
        if 0 <= s < pool:
            want[r] = ak.short_conv_step(x[r:r + 1], own[s:s + 1], weight, bias, "silu")[0]
    other = state.contiguous() if separate else None
    out = ak.short_conv_step(x, state, weight, bias, "silu", slots.cuda(), other)
    assert torch.equal(out, want) and torch.equal(other if separate else state, own)
    if separate:
        assert torch.equal(whole, kept)
    else:
        assert torch.equal(whole[:, :3], kept[:, :3])
