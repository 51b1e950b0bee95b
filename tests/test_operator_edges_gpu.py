"""Ends of the range that the documentation of the operators allows."""
import pytest
import torch

import ascend_kernel as ak
from operator_checks import conv_plain
from test_operator_overlap_cpu import hazard, small_views

pytestmark = pytest.mark.gpu


def rnd(*shape):
    return torch.randn(*shape, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "silu"])
def test_convolution_gradients_of_what_is_not_finite(act, dtype):
    """Infinities and NaN in x, with upstream gradients of zero there and elsewhere: NaN where the definition has NaN (zero times
    a derivative that is none) and nowhere else."""
    b, l, c, w = 2, 40, 16, 4
    x, weight, bias, initial = rnd(b, l, c).to(dtype), rnd(c, w), rnd(c), rnd(b, w - 1, c).to(dtype)
    x[0, 7, 1], x[0, 21, 2], x[1, 39, 3], x[1, 0, 4], initial[0, 1, 5] = float("inf"), float("nan"), float("-inf"), float("inf"), float("nan")
    dout = rnd(b, l, c).to(dtype)
    dout[:, ::2] = 0
    dout[:, 18:28] = 0

    def gradients(call, *tensors):
        leaves = [t.detach().requires_grad_(True) for t in tensors]
        return torch.autograd.grad(call(*leaves), leaves, dout.to(leaves[0].dtype))

    got = gradients(lambda x, w, b, s: ak.short_conv(x, w, b, act, s), x, weight, bias, initial)
    want = gradients(lambda x, w, b, s: conv_plain(x, w, b, act, s)[0], *(t.double() for t in (x, weight, bias, initial)))
    clean = gradients(lambda x, w, b, s: ak.short_conv(x, w, b, act, s),
                      *(t.nan_to_num(0.25, 0.25, 0.25) for t in (x, weight, bias, initial)))
    for name, g, v, k in zip(("dx", "dweight", "dbias", "dinitial"), got, want, clean):
        assert torch.equal(g.isnan(), v.isnan()), name
        assert v.isnan().any() or act is None, name
    assert torch.equal(got[0][..., 6:], clean[0][..., 6:]) and torch.equal(got[1][6:], clean[1][6:])


def test_convolution_gradients_stay_within_their_sequence():
    """An infinity in the last inputs of a packed sequence, whose gradients end there."""
    c, lengths = 16, [11, 1, 17, 24]
    x, weight, bias, dout = rnd(1, sum(lengths) + 3, c), rnd(c, 4), rnd(c), rnd(1, sum(lengths) + 3, c)
    cu = torch.tensor([0] + lengths).cumsum(0).to("cuda", torch.int32)
    results = []
    for spoil in (False, True):
        leaf = x.clone()
        if spoil:
            leaf[:, 10], leaf[:, 11], leaf[:, 52] = float("inf"), float("nan"), float("inf")
        leaf.requires_grad_(True)
        results.append(torch.autograd.grad(ak.short_conv(leaf, weight, bias, "silu", cu_seqlens=cu), leaf, dout)[0])
    good, bad = results
    for own in (slice(0, 7), slice(12, 29), slice(29, 49), slice(53, 56)):
        assert torch.equal(good[:, own], bad[:, own])
    assert bad[:, 7:12].isnan().any(-1).all() and not bad[:, 53:].any()


@pytest.mark.parametrize("b,l", [(2, 0), (0, 5), (0, 0)])
def test_gradients_of_calls_without_tokens(b, l):
    """Every tensor has its gradient: zeros for what nothing depends on, the states' own for what passes through."""
    c, w, n = 16, 4, 8
    x, weight, bias, initial = (t.requires_grad_(True) for t in (rnd(b, l, c), rnd(c, w), rnd(c), rnd(b, w - 1, c)))
    out, final = ak.short_conv(x, weight, bias, "silu", initial, return_final_state=True)
    grads = torch.autograd.grad([out, final], [x, weight, bias, initial], [torch.ones_like(out), 2 * torch.ones_like(final)])
    assert [g.shape for g in grads] == [t.shape for t in (x, weight, bias, initial)]
    assert not grads[1].any() and not grads[2].any() and (grads[3] == 2).all() and torch.equal(final, initial)
    assert not torch.autograd.grad(ak.short_conv(x, weight).sum(), weight)[0].any()
    alone = ak.short_conv(x.detach(), weight, None, None, return_final_state=True)[1]
    assert not torch.autograd.grad(alone.sum(), weight)[0].any() and not alone.any()

    tensors = [rnd(b, l, c), rnd(b, l, c), -rnd(c, n).abs(), rnd(b, l, 1, n), rnd(b, l, 1, n), rnd(c), rnd(b, l, c), rnd(c), rnd(b, c, n)]
    for t in tensors:
        t.requires_grad_(True)
    out, final = ak.selective_scan(*tensors[:8], True, tensors[8], return_final_state=True)
    grads = torch.autograd.grad([out, final], tensors, [torch.ones_like(out), 2 * torch.ones_like(final)])
    assert [g.shape for g in grads] == [t.shape for t in tensors]
    assert not any(g.any() for g in grads[:8]) and (grads[8] == 2).all() and torch.equal(final, tensors[8])
    out, final = ak.selective_scan(*tensors[:5], return_final_state=True)
    assert not final.any() and not torch.autograd.grad(out.sum() + final.sum(), tensors[2])[0].any()


def overlapping(pool):
    """(state, state_out) that share memory but are not the same slots."""
    n, inner = pool.shape[0], pool[0].numel()
    flat = pool.view(n, inner)
    shifted = torch.as_strided(flat, pool[1:].shape, pool.stride(), inner // 2)
    return [(pool[:-1], pool[1:]), (pool[1:], pool[:-1]), (pool[:-1], shifted), (pool[:2], pool[1:4:2])]


def apart(pool):
    """(state, state_out) that lie in one cache side by side, or are the same."""
    n = pool.shape[0]
    return [(pool, pool), (pool[::2], pool[1::2]), (pool[1::2], pool[::2]), (pool[:n // 2], pool[n // 2:]), (pool[::2], pool[::2]),
            (pool[:4:2], pool[:2])]


def test_state_out_that_overlaps_the_state_in_part():
    """Rows run at the same time, so that one's new state would be another's old one or not, by chance."""
    c, w, n = 8, 4, 16
    for state, out in overlapping(rnd(6, w - 1, c)):
        with pytest.raises(RuntimeError, match="short_conv_step: state_out must be state or lie apart from it"):
            ak.short_conv_step(rnd(state.shape[0], c), state, rnd(c, w), state_out=out)
    for state, out in apart(rnd(6, w - 1, c)):
        x, weight, fresh = rnd(state.shape[0], c), rnd(c, w), torch.zeros_like(state)
        want = ak.short_conv_step(x, state, weight, state_out=fresh)
        assert torch.equal(ak.short_conv_step(x, state, weight, state_out=out), want) and torch.equal(out, fresh)

    def arguments(r):
        return rnd(r, c), rnd(r, c), -rnd(c, n).abs(), rnd(r, 1, n), rnd(r, 1, n)

    for state, out in overlapping(rnd(6, c, n)):
        with pytest.raises(RuntimeError, match="selective_scan_step: state_out must be state or lie apart from it"):
            ak.selective_scan_step(*arguments(state.shape[0]), state, state_out=out)
    for state, out in apart(rnd(6, c, n)):
        a, fresh = arguments(state.shape[0]), torch.zeros_like(state)
        want = ak.selective_scan_step(*a, state, state_out=fresh)
        assert torch.equal(ak.selective_scan_step(*a, state, state_out=out), want) and torch.equal(out, fresh)


def test_every_pair_of_views_of_a_small_cache():
    """What is refused is refused before any launch; the rest gives what separate caches give."""
    weight = rnd(1, 4)
    for state, out in small_views(torch.randn(60, device="cuda")):
        rows = state.shape[0]
        state, out, x = state.view(rows, 3, 1), out.view(rows, 3, 1), rnd(rows, 1)
        if hazard(state, out):
            with pytest.raises(RuntimeError, match="state_out must be state or lie apart from it"):
                ak.short_conv_step(x, state, weight, state_out=out)
        else:
            fresh = torch.empty(rows, 3, 1, device="cuda")
            want = ak.short_conv_step(x, state.clone(), weight, state_out=fresh)
            assert torch.equal(ak.short_conv_step(x, state, weight, state_out=out), want) and torch.equal(out, fresh)


def test_sizes_that_the_records_cannot_hold():
    """2^32 + 5 rows (all at one place): as a 32-bit number they would be five."""
    rows, c, n = 2 ** 32 + 5, 1, 1
    x, weight = torch.zeros(1, 1, c, device="cuda", dtype=torch.bfloat16).expand(rows, 1, c), rnd(c, 4)
    B, A = x.unsqueeze(2), -torch.ones(c, n, device="cuda")
    slots = torch.zeros(1, device="cuda", dtype=torch.int32)
    with torch.no_grad():
        for call in (lambda: ak.short_conv(x, weight), lambda: ak.selective_scan(x, x, A, B, B)):
            with pytest.raises(RuntimeError, match="out of range"):
                call()
        cache = torch.empty(rows, 1, c, device="cuda", dtype=torch.bfloat16)  # more slots than there are numbers for them
        with pytest.raises(RuntimeError, match="short_conv_step: .*out of range"):
            ak.short_conv_step(x[:1, 0], cache, rnd(c, 2), slots=slots)
