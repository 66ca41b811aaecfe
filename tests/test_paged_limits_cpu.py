"""Sizes at the edge of what the paged KV-cache operators take: refused by the host, before anything is launched."""
import ctypes as C

import pytest

from rcutetts_b200 import _lib
from test_paged_cpu import call, pack


@pytest.mark.parametrize("page", [8, 16, 32, 64])
def test_attention_refuses_lengths_whose_last_tile_passes_31_bits(page):
    """Keys go by in tiles of up to 128: a length's last tile has to end below 2^31, or the count of tiles wraps round."""
    most = (2**31 - 128) // page
    over = dict(h=1, heads=4, qld=4 * 64, old=4 * 64, n=100, p=page)
    for pages in (most + 1, (2**31 - 1) // page):
        args = pack("attention", pages=pages, tld=pages, **over)
        assert call("ctts_op_paged_attention", args)[0] == _lib.ERR_RANGE
        assert _lib.load().ctts_op_paged_attention_workspace(args, C.byref(C.c_size_t())) == _lib.ERR_RANGE
    assert call("ctts_op_paged_attention", pack("attention", pages=most, tld=most, rows=0, **over))[0] == 0


@pytest.mark.parametrize("over", [dict(rows=2**30 + 1), dict(rows=2**31 - 1), dict(cap=2**30 + 1), dict(cap=2**31 - 1)])
def test_plan_refuses_lists_whose_loops_pass_31_bits(over):
    """The lists are filled in strides of the grid (some 75 thousand entries): a counter near 2^31 would wrap round to negative entries."""
    far = dict(pos=1 << 40, slots=1 << 41, free=1 << 42)  # lists that overlap nothing
    assert call("ctts_op_paged_plan", pack("plan", **far, **over))[0] == _lib.ERR_RANGE


@pytest.mark.parametrize("batch", [2**30 + 1, 2**31 - 1])
def test_attention_refuses_batches_whose_scan_passes_31_bits(batch):
    """Each block scans the requests in strides of its threads: near 2^31 that counter would wrap round and never end."""
    args = pack("attention", batch=batch, pages=1, tld=1)
    assert call("ctts_op_paged_attention", args)[0] == _lib.ERR_RANGE
    assert _lib.load().ctts_op_paged_attention_workspace(args, C.byref(C.c_size_t())) == _lib.ERR_RANGE
