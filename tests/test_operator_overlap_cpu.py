"""state_out of the generation steps against state, by enumeration of every byte: which pairs of views of one cache are refused."""
import itertools

import pytest
import torch

import ascend_kernel as ak
from ascend_kernel import _operands
from test_operator_refusals_cpu import Fake, fake, refused


def hazard(state, out):
    """Whether a slot of `out` shares memory with another slot of `state`, or with its own but for being the same."""
    def places(t, i):
        first = t[i].storage_offset()
        return set(range(first, first + t[i].numel()))

    return any(places(state, k) & places(out, i) and places(state, k) != places(out, i) or
               (k != i and places(state, k) & places(out, i))
               for i, k in itertools.product(range(state.shape[0]), repeat=2))


def small_views(flat):
    """Pairs of caches [n, 3] in 60 numbers."""
    inner = 3
    views = [flat.as_strided((n, inner), (step, 1), first)
             for n in (1, 2, 4) for step in (3, 4, 6, 7) for first in (0, 1, 2, 3, 6, 9, 12, 30)
             if first + (n - 1) * step + inner <= flat.numel()]
    return [(a, b) for a, b in itertools.product(views, repeat=2) if a.shape == b.shape]


def test_every_pair_of_views_of_a_small_cache():
    refusals, pairs = 0, small_views(torch.zeros(60))
    for state, out in pairs:
        try:
            _operands.apart("op", state, out)
            refuse = False
        except RuntimeError:
            refuse = True
        assert refuse == hazard(state, out), (state.shape, state.stride(), state.storage_offset(), out.stride(), out.storage_offset())
        refusals += refuse
    assert len(pairs) / 10 < refusals < len(pairs)
    _operands.apart("op", torch.zeros(0, 3), torch.zeros(0, 3))


@pytest.mark.parametrize("shift", [1, 2])
def test_words(shift):
    c, n = 8, 16
    pool = torch.zeros(6, 3, c)
    state, out = (t.as_subclass(Fake) for t in (pool[:-shift], pool[shift:]))
    refused("short_conv_step: state_out must be state or lie apart from it", ak.short_conv_step, fake(6 - shift, c), state, fake(c, 4),
            state_out=out)
    pool = torch.zeros(6, c, n)
    state, out = (t.as_subclass(Fake) for t in (pool[:-shift], pool[shift:]))
    r = 6 - shift
    refused("selective_scan_step: state_out must be state or lie apart from it", ak.selective_scan_step, fake(r, c), fake(r, c),
            fake(c, n), fake(r, 1, n), fake(r, 1, n), state, state_out=out)
