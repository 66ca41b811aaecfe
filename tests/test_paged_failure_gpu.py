"""Waits of the paged attention kernels that run out, without a GPU fault: with the error-path switch on, the first CTA never
hands a stage of its key tiles back, so its copies wait for one that stays full and give up after a thousand tries (about 1.5 ms)."""
import time

import pytest
import torch

from rcutetts_b200 import _lib
from test_paged_gpu import TYPES, Case

pytestmark = pytest.mark.gpu


def faulty(c):
    """c's output with the switch on, and the seconds that took."""
    lib = _lib.load()
    out = torch.zeros_like(c.q)
    torch.cuda.synchronize()
    assert lib.ctts_debug_inject_wait_fault(1, 1 << 10) == 0
    try:
        began = time.time()
        c.run(out=out)
        torch.cuda.synchronize()
        return out, time.time() - began
    finally:
        assert lib.ctts_debug_inject_wait_fault(0, 0) == 0


def long_requests(new, hd, q_t, kv_t):
    """Each CTA has more key tiles than stages."""
    return Case([20000] * 8, [new] * 8, 8, 4, hd, 64, q_t, kv_t, seed=30)


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 70])
def test_a_wait_that_runs_out_ends_the_call(q_t, kv_t, hd, new):
    """Within the limit's time, whatever copies were in flight; then the same calls give the same bits."""
    c = long_requests(new, hd, q_t, kv_t)
    want = c.run()
    _, took = faulty(c)
    assert took < 2.0
    assert torch.equal(c.run(), want)


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 70])
def test_what_a_wait_that_runs_out_leaves_is_nan(q_t, kv_t, hd, new):
    """A row is what it is without the fault, or NaN: never what happened to lie in a stage, and never what the output held."""
    c = long_requests(new, hd, q_t, kv_t)
    want = c.run()
    out, _ = faulty(c)
    lost = torch.isnan(out)
    assert lost[:new].any()  # the first CTA begins with the first request
    assert torch.equal(out[~lost], want[~lost]) and not lost[-new:].any()
    rows = lost.view(out.shape[0], -1, hd)
    assert torch.equal(rows.any(-1), rows.all(-1))  # a head's row as a whole
