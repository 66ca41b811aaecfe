"""Calls of the paged KV-cache operators that a server makes beside the plain ones: whole steps captured and replayed, streams of
every kind, shared pages, many heads and requests, and lengths that the device has to cut."""
import random

import pytest
import torch

from rcutetts_b200 import paged
from test_paged_gpu import BF16, F32, TYPES, Case, ints, plan_ref

pytestmark = pytest.mark.gpu


class Server:
    """Buffers of one layer's serving steps; unwritten slots hold NaN."""

    def __init__(self, batch, heads, kv, hd, p, n_pages, width, max_rows, max_new, q_t, kv_t):
        self.heads, self.kv, self.hd, self.p, self.max_rows, self.max_new, self.width = heads, kv, hd, p, max_rows, max_new, width
        self.k, self.v = (torch.full((n_pages, p, kv, hd), float("nan"), dtype=kv_t, device="cuda") for _ in range(2))
        self.tables = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(n_pages, generator=torch.Generator("cuda").manual_seed(4), device="cuda").int()
        self.ctx, self.new, self.count = ints([0] * batch), ints([0] * batch), ints([n_pages, 0, 0, 0])
        self.x = torch.full((max_rows, (heads + 2 * kv) * hd), float("nan"), dtype=q_t, device="cuda")
        self.q = torch.full((max_rows, heads, hd), 7.0, dtype=q_t, device="cuda")
        self.out = torch.full((max_rows, heads, hd), 5.0, dtype=q_t, device="cuda")
        self.gain = (1 + torch.arange(hd, device="cuda") / hd), (2 - torch.arange(hd, device="cuda") / hd)

    def step(self, stream=None):
        s = paged.paged_plan(self.ctx, self.new, self.tables, self.free, self.count, self.p, self.max_rows, stream=stream)
        paged.paged_append(self.x, self.k, self.v, s.positions, s.slots, self.heads, q_norm=self.gain[0], k_norm=self.gain[1], out=self.q, stream=stream)
        paged.paged_attention(self.q, self.k, self.v, self.tables, s.cu_rows, s.seq_lens, self.max_new, out=self.out, stream=stream)
        return s

    def state(self):
        return [t.clone() for t in (self.k, self.v, self.tables, self.free, self.ctx, self.count, self.q, self.out)]

    def load(self, new, seed):
        n = sum(max(i, 0) for i in new)
        self.new.copy_(ints(new))
        self.x.fill_(float("nan"))  # rows of padding
        self.x[:n] = torch.randn(n, self.x.shape[1], generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(self.x.dtype)

    def advance(self, s):
        self.ctx.copy_(s.seq_lens)
        self.count.copy_(s.state)


STEPS = [[37, 5, 0, 60], [1, 40, 70, 1], [1, 1, 1, 1], [20, -1, 1, 1], [1, 33, 1, -1], [1, 1, 1, 0], [1, 1, 90, 16], [0, 0, 0, 0], [-1, -1, -1, -1], [3, 0, 2, 1]]


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("heads, kv, hd", [(12, 4, 64), (16, 8, 128)])
def test_a_captured_step_serves_many(q_t, kv_t, heads, kv, hd):
    """plan, append and attention in one graph, replayed over admissions, growth, idle and finished requests: what the same calls
    give eagerly, bit for bit, and rows of padding untouched."""
    shape = (4, heads, kv, hd, 16, 40, 14, 160, 90, q_t, kv_t)
    eager, graphed = Server(*shape), Server(*shape)
    graph = torch.cuda.CUDAGraph()
    graphed.load([0] * 4, 0)
    graphed.step()  # what the first calls set up
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        s = graphed.step()
    for i, new in enumerate(STEPS):
        eager.load(new, i)
        graphed.load(new, i)
        eager.out.fill_(5.0)
        graphed.out.fill_(5.0)
        want = plan_ref(eager.ctx.tolist(), new, eager.tables.tolist(), eager.free.tolist(), int(eager.count[0]), 16, 160)
        e = eager.step()
        graph.replay()
        assert [t.tolist() for t in (eager.tables, eager.free, *e)] == list(want)
        assert all(torch.equal(a, b) for a, b in zip(e, s))
        rows = int(e.state[1])
        assert (graphed.out[rows:] == 5.0).all() and torch.isfinite(graphed.out[:rows]).all()
        eager.advance(e)
        graphed.advance(s)
        for a, b in zip(eager.state(), graphed.state()):
            assert torch.equal(a.nan_to_num(3e3), b.nan_to_num(3e3))


def test_streams_of_every_kind():
    """The default stream beside another current one, an external stream, an address: outputs belong to the stream that made them."""
    a, b = (Server(4, 12, 4, 64, 16, 40, 14, 160, 90, F32, BF16) for _ in range(2))
    side = torch.cuda.Stream()
    kinds = [torch.cuda.default_stream(), side, side.cuda_stream, torch.cuda.ExternalStream(side.cuda_stream), None, 0]
    torch.cuda.synchronize()
    for i, new in enumerate(STEPS):
        a.load(new, i)
        b.load(new, i)
        torch.cuda.synchronize()
        a.advance(a.step())
        with torch.cuda.stream(torch.cuda.Stream()):
            s = b.step(stream=kinds[i % len(kinds)])
            torch.cuda.synchronize()
            b.advance(s)
            torch.cuda.synchronize()
        for x, y in zip(a.state(), b.state()):
            assert torch.equal(x.nan_to_num(3e3), y.nan_to_num(3e3))


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("new", [1, 50])
def test_shared_pages(q_t, kv_t, new):
    """A page may stand in several tables, and twice in one (a prefix of many requests)."""
    c = Case([160] * 6, [new] * 6, 4, 2, 64, 16, q_t, kv_t, seed=2)
    c.tables[1:, :8] = c.tables[0, :8]
    c.tables[3, 2] = c.tables[3, 5]
    c.tables[4, :8] = c.tables[4, 0].clone()
    c.check(c.run())


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("heads, kv, hd", [(64, 64, 64), (128, 32, 128), (1024, 1024, 64)])
def test_many_heads(q_t, kv_t, heads, kv, hd):
    for new in (1, 20):
        c = Case([70, 0, 300], [new] * 3, heads, kv, hd, 16, q_t, kv_t, seed=3)
        out = c.run()
        some = slice(0, kv, max(1, kv // 8))  # a few KV heads of all
        g = heads // kv
        pick = torch.arange(kv)[some]
        c.q, out = (t.view(-1, kv, g, hd)[:, pick].flatten(1, 2) for t in (c.q, out))
        c.k, c.v, c.heads, c.kv = c.k[:, :, pick], c.v[:, :, pick], len(pick) * g, len(pick)
        c.check(out)


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("most", [1, 30])
def test_a_batch_of_twenty_thousand(q_t, kv_t, most):
    rng = random.Random(6)
    n = 20000
    lens = [rng.choice([0, rng.randint(1, 40)]) for _ in range(n)]
    new = [min(x, rng.choice([0, 1, 1, 1, most])) for x in lens]
    c = Case([x - y for x, y in zip(lens[:50], new[:50])], new[:50], 2, 1, 64, 16, q_t, kv_t, seed=7)  # pages of the first fifty
    pick = [rng.randrange(50) for _ in range(n)]
    rows = torch.cat([torch.arange(int(c.cu[b]), int(c.cu[b + 1]), device="cuda") for b in pick])
    alone = c.run(max_new=most)
    c.check(alone)
    cu = torch.tensor([0] + [new[b] for b in pick]).cumsum(0).int().cuda()
    at = torch.tensor(pick, device="cuda")
    out = paged.paged_attention(c.q[rows].contiguous(), c.k, c.v, c.tables[at].contiguous(), cu, c.lens[at].contiguous(), most, scale=c.scale)
    # other requests share the GPU, so the cuts are others: within what divided sums move
    tol = 2.0**-7 if q_t == BF16 else 2.0**-18
    assert ((out.float() - alone[rows].float()).abs() <= tol * c.v.float().nan_to_num(0).abs().amax()).all()


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("new", [1, 40])
def test_rows_that_do_not_begin_at_zero(q_t, kv_t, new):
    c = Case([30, 200], [new] * 2, 4, 2, 64, 16, q_t, kv_t, seed=9)
    want = c.run()
    q = torch.full((c.total + 9, 4, 64), float("nan"), dtype=q_t, device="cuda")
    q[4: 4 + c.total] = c.q
    out = torch.full_like(q, 2.0)
    paged.paged_attention(q, c.k, c.v, c.tables, c.cu + 4, c.lens, new, scale=c.scale, out=out)
    assert torch.equal(out[4: 4 + c.total], want) and (out[:4] == 2.0).all() and (out[4 + c.total:] == 2.0).all()


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("new", [1, 40])
def test_lengths_are_cut_to_what_the_buffers_hold(q_t, kv_t, new):
    """Lengths beyond the table count as the table's, row offsets are cut to the rows there are, backward ones give no rows."""
    c = Case([30, 200, 64], [new] * 3, 4, 2, 64, 16, q_t, kv_t, seed=10, spare_cols=0)
    width = c.tables.shape[1]
    c.tables[:, :] = c.tables[1]  # every entry is a page with keys
    c.lens[1] = width * 16
    page = int(c.tables[1, width - 1])
    c.k[page], c.v[page] = c.k[page].nan_to_num(0.5), c.v[page].nan_to_num(0.5)
    c.ctx[1] = width * 16 - new
    c.ctx[2] = 64
    full = c.run()
    c.check(full)
    lens, cu = c.lens.clone(), c.cu.clone()
    c.lens[1] = 2**31 - 1
    assert torch.equal(c.run(), full)

    def check_first_two(out):
        """The cuts follow from all lengths, so where another request's changed the bits may: each is held to 64 bits."""
        c.new = [new, new, 0]
        c.check(out)
        c.new = [new] * 3

    c.lens[1], c.lens[2] = lens[1], -(2**31)
    out = c.run()
    check_first_two(out)
    assert (out[2 * new:] == 0).all()
    c.lens.copy_(lens)
    c.cu[3] = 2**31 - 1
    assert torch.equal(c.run(), full)
    c.cu[0], c.cu[3] = -7, -(2**31)  # the first request begins where the rows do, the last has none
    out = c.run(out=torch.full_like(c.q, 8.0))
    c.cu[0] = 0
    check_first_two(out)
    assert (out[2 * new:] == 8.0).all()
    c.cu.copy_(cu)
    assert torch.equal(c.run(), full)
