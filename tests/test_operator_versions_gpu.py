"""The generation steps write a cache in place, as the framework's own in-place operations do: what was saved of it for a
backward pass counts as changed, whichever view of the cache was written."""
import pytest
import torch

import ascend_kernel as ak

pytestmark = pytest.mark.gpu

C, W, N = 24, 4, 8


def cache(*inner):
    """One layer's share [slots, ...] of a cache of three layers, and the whole cache."""
    whole = torch.randn(5, 3, *inner, device="cuda")
    return whole[:, 1], whole


def conv_step(state, state_out=None):
    slots = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        ak.short_conv_step(torch.randn(2, C, device="cuda"), state, torch.randn(C, W, device="cuda"), None, "silu", slots, state_out)


def scan_step(state, state_out=None):
    slots = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    rnd = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    with torch.no_grad():
        ak.selective_scan_step(rnd(2, C), rnd(2, C), -rnd(C, N).abs(), rnd(2, 1, N), rnd(2, 1, N), state, dt_softplus=True,
                               slots=slots, state_out=state_out)


STEPS = [(conv_step, (W - 1, C)), (scan_step, (C, N))]


@pytest.mark.parametrize("step,inner", STEPS)
def test_a_step_counts_as_a_change_of_what_it_writes(step, inner):
    state, whole = cache(*inner)
    before = whole._version
    step(state)
    assert whole._version == before + 1 and state._version == before + 1
    out, other = cache(*inner)
    written, read = other._version, whole._version
    step(state, out)
    assert other._version == written + 1 and whole._version == read


@pytest.mark.parametrize("step,inner", STEPS)
def test_saved_by_the_frameworks_own_operation(step, inner):
    state, whole = cache(*inner)
    leaf = torch.randn(inner, device="cuda", requires_grad=True)
    product = (state * leaf).sum()
    step(state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


def test_initial_state_of_the_convolution():
    """Its backward reads the initial state again."""
    state, weight = torch.randn(5, W - 1, C, device="cuda"), torch.randn(C, W, device="cuda", requires_grad=True)
    x = torch.randn(5, 9, C, device="cuda")
    out = ak.short_conv(x, weight, None, "silu", state)
    conv_step(state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), weight)
    out = ak.short_conv(x, weight, None, "silu", state)
    conv_step(state, state.clone())  # writes another one
    torch.autograd.grad(out.sum(), weight)


def test_initial_state_of_the_scan():
    state = torch.randn(5, C, N, device="cuda")
    rnd = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    x = rnd(5, 9, C).requires_grad_(True)
    out = ak.selective_scan(x, rnd(5, 9, C), -rnd(C, N).abs(), rnd(5, 9, 1, N), rnd(5, 9, 1, N), dt_softplus=True, initial_states=state)
    scan_step(state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), x)


@pytest.mark.parametrize("step,inner", STEPS)
def test_caches_of_inference_mode(step, inner):
    """They have no version; a step takes them inside the mode and outside of it."""
    with torch.inference_mode():
        state, _ = cache(*inner)
        kept = state.clone()
        step(state)
        assert not torch.equal(state, kept)
    kept = state.clone()
    step(state)
    assert not torch.equal(state, kept)


def test_a_cache_for_new_states_that_requires_gradients():
    x, state, weight = torch.randn(2, C, device="cuda"), torch.randn(2, W - 1, C, device="cuda"), torch.randn(C, W, device="cuda")
    rnd = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    leaf = torch.zeros_like(state).requires_grad_(True)
    with pytest.raises(RuntimeError, match="short_conv_step: has no gradients"):
        ak.short_conv_step(x, state, weight, state_out=leaf)
    states = rnd(2, C, N)
    with pytest.raises(RuntimeError, match="selective_scan_step: has no gradients"):
        ak.selective_scan_step(x, rnd(2, C), -rnd(C, N).abs(), rnd(2, 1, N), rnd(2, 1, N), states,
                               state_out=torch.zeros_like(states).requires_grad_(True))
    with torch.no_grad():
        ak.short_conv_step(x, state, weight, state_out=leaf)
    assert leaf.any()
