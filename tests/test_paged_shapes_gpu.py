"""Paged attention at shapes beside those of test_paged_gpu: 128 dims in runs of 9 to 16 packed rows, over every page size and
order, and rows behind a max_new that cuts requests."""
import pytest
import torch

from test_paged_gpu import BF16, TYPES, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads, kv, new", [(6, 2, 2), (6, 2, 3), (6, 2, 5), (16, 1, 1), (16, 2, 2), (5, 1, 2), (5, 1, 3), (9, 1, 1), (11, 1, 1), (4, 2, 8), (13, 13, 9)])
def test_short_runs_of_both_head_sizes(q_t, kv_t, hd, heads, kv, new):
    """4 to 16 packed rows, 9 and 16 among them; a request that cuts divide, and missing pages."""
    c = Case([0, 40, 129, 63, 9000, 300], [new, 1, new, max(1, new - 1), new, new], heads, kv, hd, 16, q_t, kv_t, seed=new + heads)
    dead = [(2, 4), (4, 0), (4, 300), (5, 18)]
    for b, col in dead:
        c.tables[b, col] = -1
    out = c.run()
    c.check(out, dead)
    assert torch.equal(out, c.run())
    short = Case([21, 0, 90] * 150, [new] * 450, heads, kv, hd, 16, q_t, kv_t, seed=new)  # whole items
    out = short.run()
    short.ctx, short.new = short.ctx[:9], short.new[:9]
    short.check(out)


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("p", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_page_sizes_and_layouts_of_128_dims(q_t, kv_t, p, layout):
    one = Case([0, p - 1, p, 3 * p + 1, 500], [1] * 5, 4, 2, 128, p, q_t, kv_t, layout, seed=p)
    one.check(one.run())
    run = Case([0, p - 1, p, 3 * p + 1, 500], [6] * 5, 4, 2, 128, p, q_t, kv_t, layout, seed=p + 1)
    run.check(run.run())
    many = Case([0, p, 3 * p + 1, 500, 0], [2 * p + 3, 40, 1, 77, p], 4, 2, 128, p, q_t, kv_t, layout, seed=p + 2)
    many.check(many.run())


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cut", [1, 7, 20, 70])
def test_rows_ahead_of_a_cut_are_exact(q_t, kv_t, hd, cut):
    c = Case([30, 100, 700, 5], [90, 3, 130, 1], 4, 2, hd, 16, q_t, kv_t, seed=cut)
    full = c.run()
    c.check(full)
    out = torch.full_like(c.q, 9.0)
    c.run(out=out, max_new=cut)
    for b, n in enumerate(c.new):
        at = int(c.cu[b])
        assert (out[at + min(n, cut): at + n] == 9.0).all()
        out[at + min(n, cut): at + n] = full[at + min(n, cut): at + n]
    c.check(out)  # the rows ahead of the cut, against 64 bits
