"""Sizes at the far end of what the entry points take, by what they report: nothing is allocated or launched."""
import ctypes

import pytest
import torch

from ascend_kernel import _capi

NONE = ctypes.addressof(ctypes.create_string_buffer(16))


@pytest.mark.skipif(torch.cuda.is_available(), reason="without a device no sequence is cut into segments")
@pytest.mark.parametrize("tokens", [2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, 2 ** 30 + 64, 2 ** 31 - 2 ** 21])
@pytest.mark.parametrize("rows", [1, 200])
def test_a_sequence_that_is_not_cut_is_one_item(rows, tokens):
    """The gradients' workspace has dB and dC of every token (one block of channels) and a row of dstate + 2 numbers per channel
    for each item.  An item that does not begin a sequence would begin from its initial state."""
    channels, n = 2, 3
    args = _capi.SsdScanArgs(x=NONE, dt=NONE, bm=NONE, cm=NONE, A=NONE, tokens=tokens, rows=rows, channels=channels, dstate=n, groups=1)
    floats = _capi.lib.ssd_selective_scan_grad_work_bytes(ctypes.byref(args)) // 4
    items = (floats - 2 * rows * tokens * n) / ((n + 2) * channels)
    assert items == rows
