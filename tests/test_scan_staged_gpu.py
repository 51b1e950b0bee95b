"""selective_scan where warps of their own stage its tiles (sequences, or segments of them, of 256 tokens and more), in all layouts,
types and passes, with activations that are aligned column slices; and its gradients where sequences are not cut into
segments.  Which of them a size reaches is asked of the library's workspace sizes, and asserted.

Bounds are those of test_selective_scan_gpu.py."""
import ctypes

import pytest
import torch

import ascend_kernel as ak
from ascend_kernel import _capi
from operator_checks import near, scan_plain
from test_selective_scan_gpu import double, flush, magnitudes, make, plain_gradients, rounding_count

pytestmark = pytest.mark.gpu

F32, BF16, F16 = DTYPES = [torch.float32, torch.bfloat16, torch.float16]
STAGED = 256  # tokens from which on warps of their own stage the tiles


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def segments(rows, tokens, channels, n, groups, packed, gradients):
    """Into how many items the sequences are cut (rows, or the packed ones' numbering, where they are not)."""
    here = ctypes.addressof(ctypes.create_string_buffer(16))
    a = _capi.SsdScanArgs(x=here, dt=here, bm=here, cm=here, A=here, tokens=tokens, rows=rows, channels=channels, dstate=n, groups=groups,
                          cu_seqlens=here if packed else None)
    if not gradients:
        floats = _capi.lib.ssd_selective_scan_work_bytes(ctypes.byref(a)) // 4
        return floats // (channels * (n + 1)) if floats else None
    floats = _capi.lib.ssd_selective_scan_grad_work_bytes(ctypes.byref(a)) // 4
    per_group = (channels // groups + 63) // 64
    floats -= 2 * per_group * tokens * (1 if packed else rows) * groups * n
    whole = rows + 1 if packed else rows
    if floats == whole * (n + 2) * channels:
        return None
    items = floats // (channels * (2 * n + 3))
    assert (items * channels * (n + 1) + 3) // 4 * 4 + items * (n + 2) * channels == floats
    return items


def aligned_slices(tensors, widths=(0, 1, 3, 4, 6)):
    """x, dt, B, C and z as column slices of one wider projection, every one at a multiple of four columns."""
    parts = [t.flatten(2) for i, t in enumerate(tensors) if i in widths and t is not None]
    pad = torch.zeros_like(parts[0][..., :4])
    wide = torch.cat([pad] + [p for part in parts for p in (part, pad[..., :4 + -part.shape[-1] % 4])], -1)
    at, out = 4, []
    for i, t in enumerate(tensors):
        if i not in widths or t is None:
            out.append(t)
            continue
        size = t[0, 0].numel()
        out.append(wide[..., at:at + size].unflatten(-1, t.shape[2:]))
        at += size + 4 + -size % 4
        assert torch.equal(out[-1], t) and not out[-1].is_contiguous()
    return out


def check_scan(tensors, l, what):
    x, dt, A, B, C, D, z, bias, initial = tensors
    out, final = ak.selective_scan(x, dt, A, B, C, D, z, bias, True, initial, return_final_state=True)
    want, last = scan_plain(*map(double, (x, dt, A, B, C, D, z, bias)), True, double(initial))
    top, top_h = magnitudes(x, dt, A, B, C, D, z, bias, True, initial)
    near(out, want, top, rounding_count(l), f"out {what}", flush(l))
    near(final, last, top_h, rounding_count(l), f"final {what}", flush(l))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,n,g", [(9, 8, 1), (10, 8, 1), (9, 12, 2), (9, 16, 1), (10, 16, 4), (9, 32, 1), (9, 28, 1), (9, 64, 1), (9, 36, 2)])
@pytest.mark.parametrize("gated,sliced", [(True, False), (True, True), (False, True)])
def test_scan_with_staging_warps(b, n, g, gated, sliced, dtype):
    l, c = 263, 512
    assert segments(b, l, c, n, g, False, False) is None and l >= STAGED
    assert (b * c // 32 <= sms()) == (b == 9)  # two columns or four per warp, where there are eight
    tensors = list(make(b, l, c, n, g, dtype, seed=n))
    if not gated:
        tensors[6] = None
    check_scan(aligned_slices(tensors) if sliced else tensors, l, "staged")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,sliced", [(8, False), (16, True), (32, False), (64, True)])
def test_segments_with_staging_warps(n, sliced, dtype):
    """The pass over the segments' own end states, and the walk from the joined ones."""
    l, c = 2431, 1024
    assert segments(1, l, c, n, 1, False, False) == -(-l // 320)
    tensors = make(1, l, c, n, 1, dtype, seed=n)
    check_scan(aligned_slices(tensors) if sliced else tensors, l, "segments")


def packed_case(lengths, behind, c, n, g, dtype, seed):
    total = sum(lengths) + behind
    tensors = make(1, total, c, n, g, dtype, states=len(lengths), seed=seed)
    cu = torch.tensor([0] + lengths).cumsum(0).to("cuda", torch.int32)
    return total, aligned_slices(tensors), cu


def part_of(tensors, own, s):
    return [t[:, own] if i in (0, 1, 3, 4, 6) else t[s:s + 1] if i == 8 else t for i, t in enumerate(tensors)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,behind,c,n", [([700, 0, 1, 33, 0, 1025, 290, 600, 251, 5], 40, 512, 16),
                                                ([1500, 0, 31, 1601, 1100], 9, 448, 32)])
def test_packed_sequences_with_staging_warps(lengths, behind, c, n, dtype):
    """Not cut, and cut into segments."""
    total, tensors, cu = packed_case(lengths, behind, c, n, 1, dtype, 11)
    assert total // len(lengths) >= STAGED
    assert segments(len(lengths), total, c, n, 1, True, False) == (None if c == 512 else total // STAGED + len(lengths) + 1)
    out, final = ak.selective_scan(*tensors[:8], True, tensors[8], cu, True)
    at = 0
    for s, m in enumerate(lengths):
        own = slice(at, at + m)
        at += m
        if m == 0:
            assert torch.equal(final[s], tensors[8][s])
            continue
        part = part_of(tensors, own, s)
        want, last = scan_plain(*map(double, part[:8]), True, double(part[8]))
        top, top_h = magnitudes(*part[:8], True, part[8])
        near(out[:, own], want, top, rounding_count(m), f"out {s}", flush(m))
        near(final[s:s + 1], last, top_h, rounding_count(m), f"final {s}", flush(m))
    assert not out[:, at:].any()


def check_gradients(tensors, l, dtype):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in tensors]
    out, final = ak.selective_scan(*leaves[:8], True, leaves[8], return_final_state=True)
    dout, dfinal = torch.randn_like(out), torch.randn_like(final)
    got = iter(torch.autograd.grad([out, final], [t for t in leaves if t is not None], [dout, dfinal]))
    got = [None if t is None else next(got) for t in leaves]
    want, tops = plain_gradients([None if t is None else t.detach() for t in leaves], True, dout, dfinal)
    b, c = tensors[0].shape[0], tensors[0].shape[2]
    many = {2: b * l, 3: c, 4: c, 5: b * l, 7: b * l}
    for i, name in enumerate(("dx", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dinitial")):
        if got[i] is not None:
            near(got[i], want[i], tops[i], 2 * rounding_count(l) + 16 + many.get(i, 0), name, flush(l))


@pytest.mark.parametrize("n,dtype,gated,sliced", [(4, F32, True, False), (8, BF16, True, True), (16, F32, False, False), (16, BF16, True, True),
                                                  (16, F16, True, False), (32, F16, True, True), (64, BF16, True, False)])
def test_gradients_of_segments_with_staging_warps(n, dtype, gated, sliced):
    """Backward in time over each segment, and the gradients from the joined ones."""
    l, c = 3659, 1024
    assert segments(1, l, c, n, 1, False, True) == -(-l // STAGED)
    tensors = list(make(1, l, c, n, 1, dtype, seed=n))
    if not gated:
        tensors[6] = None
    check_gradients(aligned_slices(tensors) if sliced else tensors, l, dtype)


@pytest.mark.parametrize("n,g,dtype,gated,sliced", [(16, 1, BF16, True, True), (16, 2, F32, False, True), (24, 1, F16, True, False),
                                                    (7, 1, BF16, False, False)])
def test_gradients_of_sequences_that_are_not_cut(n, g, dtype, gated, sliced):
    b, l, c = 10, 141, 512
    assert segments(b, l, c, n, g, False, True) is None
    tensors = list(make(b, l, c, n, g, dtype, seed=n))
    if not gated:
        tensors[6] = None
    check_gradients(aligned_slices(tensors) if sliced else tensors, l, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_packed_gradients_with_staging_warps(dtype):
    lengths, behind, c, n = [1900, 0, 3, 1307, 1000], 11, 896, 8
    total, tensors, cu = packed_case(lengths, behind, c, n, 1, dtype, 12)
    assert segments(len(lengths), total, c, n, 1, True, True) == total // STAGED + len(lengths) + 1
    assert total // len(lengths) >= STAGED
    leaves = [t.detach().requires_grad_(True) for t in tensors]
    out, final = ak.selective_scan(*leaves[:8], True, leaves[8], cu, True)
    dout, dfinal = torch.randn_like(out), torch.randn_like(final)
    grads = torch.autograd.grad([out, final], leaves, [dout, dfinal])
    at, da, da_top = 0, 0, 0
    for s, m in enumerate(lengths):
        own = slice(at, at + m)
        at += m
        if m == 0:
            assert torch.equal(grads[8][s], dfinal[s])
            continue
        expected, tops = plain_gradients(part_of(tensors, own, s), True, dout[:, own], dfinal[s:s + 1])
        for i in (0, 1, 3, 4, 6):
            near(grads[i][:, own], expected[i], tops[i], 2 * rounding_count(m) + 16 + c, f"gradient {i} of {s}", flush(m))
        near(grads[8][s:s + 1], expected[8], tops[8], 2 * rounding_count(m) + 16, f"dinitial {s}", flush(m))
        da, da_top = da + expected[2], da_top + tops[2]
    near(grads[2], da, da_top, 2 * rounding_count(max(lengths)) + 16 + total, "dA", flush(total))
    assert not any(grads[i][:, at:].any() for i in (0, 1, 3, 4, 6))
