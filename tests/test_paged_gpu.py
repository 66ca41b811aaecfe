"""The paged KV-cache operators against plain implementations: the plan
against Python integers, append and attention against 64-bit arithmetic on the
same stored inputs, and a run of the three beside the LM's contiguous cache.

Tolerances count roundings.  A rounding to bf16 is off by at most 2^-8 of the
value, to float32 by 2^-24; a product sum of n float32 terms by n * 2^-24 of
the sum of their magnitudes."""
import math
import random

import numpy as np
import pytest
import torch

from rcutetts_b200 import _lib, paged
from rcutetts_b200._lib import CttsError

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def up(a, b):
    return -(-a // b)


# ------------------------------------------------------------------- plan

def plan_ref(ctx, new, tables, free, count, p, max_rows):
    """The contract, request by request."""
    tables, free, width = [list(r) for r in tables], list(free), len(tables[0])
    ctx = [max(c, 0) for c in ctx]
    top = max(0, min(count, len(free)))
    stack = free[:top]
    for b, n in enumerate(new):
        if n < 0:
            stack += tables[b][: min(up(ctx[b], p), width)]
    stack = stack[: len(free)]
    free[top: len(stack)] = stack[top:]
    lens, cu, positions, slots, taken, granted = [], [0], [], [], 0, len(ctx)
    for b, n in enumerate(new):
        held, after = up(ctx[b], p), up(ctx[b] + max(n, 0), p)
        if granted == len(ctx) and n > 0 and (after - held > len(stack) or cu[-1] + n > max_rows or after > width):
            granted = b
        rows = max(n, 0) if granted == len(ctx) else 0
        if rows:
            for col in range(held, after):
                tables[b][col] = stack.pop()
                taken += 1
            for pos in range(ctx[b], ctx[b] + rows):
                positions.append(pos)
                slots.append(tables[b][pos // p] * p + pos % p)
        lens.append(0 if n < 0 else ctx[b] + rows)
        cu.append(cu[-1] + rows)
    pad = [-1] * (max_rows - len(slots))
    return tables, free, lens, cu, positions + pad, slots + pad, [len(stack), cu[-1], granted, taken]


def run_plan(ctx, new, tables, free, count, p, max_rows):
    t, f = ints(tables), ints(free)
    s = paged.paged_plan(ints(ctx), ints(new), t, f, ints([count]), p, max_rows)
    return [x.tolist() for x in (t, f, s.seq_lens, s.cu_rows, s.positions, s.slots, s.state)]


def random_plan(rng, batch, p, ctx_hi, new_hi, spare, rows_short=0, width_short=0):
    ctx = [rng.choice([0, rng.randint(0, ctx_hi), p * rng.randint(0, ctx_hi // p)]) for _ in range(batch)]
    new = [rng.choice([-1, 0, 1, 1, rng.randint(1, new_hi)]) for _ in range(batch)]
    width = max(1, max(up(c + max(n, 0), p) for c, n in zip(ctx, new)) - width_short)
    ctx = [min(c, width * p) for c in ctx]
    held = sum(up(c, p) for c in ctx)
    cap = held + max(0, sum(up(c + n, p) - up(c, p) for c, n in zip(ctx, new) if n > 0) + spare)
    order = list(range(cap))
    rng.shuffle(order)
    tables, at = [], 0
    for c in ctx:
        k = up(c, p)
        tables.append(order[at: at + k] + [-1] * (width - k))
        at += k
    free = order[at:] + [-7] * held
    rows = max(0, sum(n for n in new if n > 0) - rows_short)
    return ctx, new, tables, free, cap - held, p, rows


@pytest.mark.parametrize("batch", [1, 2, 31, 64, 511, 513, 1500])
@pytest.mark.parametrize("p", [8, 16, 256])
def test_plan(batch, p):
    rng = random.Random(batch * 1000 + p)
    args = random_plan(rng, batch, p, 700, 300, 3)
    assert run_plan(*args) == list(plan_ref(*args))


@pytest.mark.parametrize("spare, rows_short, width_short", [(-9, 0, 0), (-10 ** 6, 0, 0), (2, 40, 0), (2, 10 ** 6, 0), (2, 0, 6), (-3, 5, 1)])
def test_plan_refuses_from_the_first_that_does_not_fit(spare, rows_short, width_short):
    for seed in range(6):
        args = random_plan(random.Random(seed), 40, 16, 300, 60, spare, rows_short, width_short)
        assert run_plan(*args) == list(plan_ref(*args))


def test_plan_widest_batch_and_many_rows():
    rng = random.Random(5)
    args = random_plan(rng, 4096, 16, 100, 90, 1)
    assert run_plan(*args) == list(plan_ref(*args))
    with pytest.raises(CttsError) as e:
        paged.paged_plan(ints([0] * 4097), ints([1] * 4097), torch.zeros(4097, 1, dtype=torch.int32, device="cuda"), ints([0]), ints([1]), 16, 9)
    assert e.value.code == _lib.ERR_RANGE


def test_plan_bad_device_values_stay_in_range():
    # a free count beyond the stack, negative lengths, huge new lengths
    assert run_plan([-5, 3], [2, 1], [[-1], [0]], [2, 1], 99, 8, 4)[2:] == [[2, 4], [0, 2, 3], [0, 1, 3, -1], [8, 9, 3, -1], [1, 3, 2, 1]]
    big = 2 ** 31 - 1
    assert run_plan([big, 3], [big, 1], [[0], [1]], [2, 3], 2, 8, 4)[2:] == [[big, 3], [0, 0, 0], [-1] * 4, [-1] * 4, [2, 0, 0, 0]]
    assert run_plan([0, 3], [1, 1], [[-1], [1]], [2, 3], -4, 8, 4)[2:] == [[0, 3], [0, 0, 0], [-1] * 4, [-1] * 4, [0, 0, 0, 0]]
    # a page number that no pool has gives no slot
    assert run_plan([3], [1], [[2 ** 30]], [0], 1, 8, 1)[5] == [-1]


def test_plan_again_gives_the_same_step():
    args = random_plan(random.Random(3), 50, 16, 300, 60, 0)
    t, f = ints(args[2]), ints(args[3])
    first = None
    for _ in range(3):
        s = paged.paged_plan(ints(args[0]), ints(args[1]), t, f, ints([args[4]]), args[5], args[6])
        now = [x.tolist() for x in (t, f, *s)]
        assert first is None or now == first
        first = now


def test_plan_tables_inside_a_wider_array():
    wide = torch.full((3, 10), -5, dtype=torch.int32, device="cuda")
    s = paged.paged_plan(ints([0, 0, 0]), ints([9, 0, 17]), wide[:, 2:5], ints([4, 5, 6, 7, 8]), ints([5]), 8, 26)
    assert s.state.tolist() == [0, 26, 3, 5]
    assert wide.tolist() == [[-5, -5, 8, 7] + [-5] * 6, [-5] * 10, [-5, -5, 6, 5, 4] + [-5] * 5]


def test_steps_of_a_serving_loop():
    """Admission, growth and release over many steps: no page is ever held twice or lost."""
    rng = random.Random(11)
    p, batch, n_pages, width = 16, 12, 60, 8
    ctx, count = ints([0] * batch), ints([n_pages])
    tables = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    free = torch.arange(n_pages, dtype=torch.int32, device="cuda")
    lens = [0] * batch
    for step in range(60):
        new = [rng.choice([0, 1, 1, rng.randint(1, 40)]) if lens[b] < 90 else -1 for b in range(batch)]
        want = plan_ref(lens, new, tables.tolist(), free.tolist(), int(count[0]), p, 64)
        s = paged.paged_plan(ctx, ints(new), tables, free, count, p, 64)
        assert [x.tolist() for x in (tables, free, s.seq_lens, s.cu_rows, s.positions, s.slots, s.state)] == list(want)
        ctx, count, lens = s.seq_lens, s.state, s.seq_lens.tolist()
        held = [pg for b in range(batch) for pg in tables[b, : up(lens[b], p)].tolist()]
        assert sorted(held + free[: int(count[0])].tolist()) == list(range(n_pages))


# ----------------------------------------------------------------- append

def pool(n, p, h, d, dtype, layout, fill=None):
    shape = (n, h, p, d) if layout == "hnd" else (n, p, h, d)
    t = torch.randn(shape, device="cuda").to(dtype) if fill is None else torch.full(shape, fill, dtype=dtype, device="cuda")
    return t.transpose(1, 2) if layout == "hnd" else t


def append_ref(x, heads, kv, hd, positions, q_norm, k_norm, eps, theta):
    x = x.double().view(x.shape[0], heads + 2 * kv, hd)
    qk, v = x[:, : heads + kv], x[:, heads + kv:]
    if q_norm is not None:
        qk = qk / torch.sqrt((qk ** 2).mean(-1, keepdim=True) + eps)
        qk = torch.cat([qk[:, :heads] * q_norm.double(), qk[:, heads:] * k_norm.double()], 1)
    ang = positions.double()[:, None] * theta ** (-torch.arange(0, hd, 2, device="cuda").double() / hd)
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    a, b = qk[..., : hd // 2], qk[..., hd // 2:]
    qk = torch.cat([a * c - b * s, a * s + b * c], -1)
    return qk[:, :heads], qk[:, heads:], v


def close_append(got, want, dtype, pair):
    # pair: magnitude of the rotated pair.  Norm: hd + 5 roundings at most on the sum, half of that under the root; sine and
    # cosine within 2^-22 (reduced angle and function); the rotation's three roundings: 2^-17 in all with room; one to the type
    tol = pair * 2.0 ** -17 + (want.abs() * 2.0 ** -8 if dtype == BF16 else 0)
    assert ((got.double() - want).abs() <= tol + 1e-30).all()


def pairs(y):
    h = y.shape[-1] // 2
    m = torch.hypot(y[..., :h], y[..., h:])
    return torch.cat([m, m], -1)


@pytest.mark.parametrize("x_t, q_t, kv_t", [(F32, F32, F32), (F32, F32, BF16), (F32, BF16, BF16), (BF16, BF16, BF16), (BF16, F32, F32)])
@pytest.mark.parametrize("heads, kv, hd, layout", [(12, 4, 64, "nhd"), (16, 8, 128, "hnd"), (1, 1, 64, "hnd"), (5, 1, 128, "nhd"), (40, 8, 64, "nhd")])
@pytest.mark.parametrize("rows, norm", [(1, True), (37, True), (37, False)])
def test_append(x_t, q_t, kv_t, heads, kv, hd, layout, rows, norm):
    torch.manual_seed(rows * hd + heads)
    p, n = 16, 9
    x = torch.randn(rows, (heads + 2 * kv) * hd, device="cuda").to(x_t)
    slots = torch.randperm(n * p, device="cuda")[:rows].int()
    positions = torch.randint(0, 100000, (rows,), device="cuda", dtype=torch.int32)
    if rows > 3:
        slots[[0, 20]] = torch.tensor([-1, n * p], dtype=torch.int32, device="cuda")  # no such slot: nothing is written
        positions[5], positions[6] = 0, 2 ** 20 + 1
    g = (1 + 0.2 * torch.randn(2, hd, device="cuda")) if norm else (None, None)
    k, v = pool(n, p, kv, hd, kv_t, layout), pool(n, p, kv, hd, kv_t, layout)
    k0, v0 = k.clone(), v.clone()
    out = torch.full((rows, heads, hd), 7.0, dtype=q_t, device="cuda")
    got = paged.paged_append(x, k, v, positions, slots, heads, q_norm=g[0], k_norm=g[1], eps=1e-6, theta=1e6, out=out)
    assert got is out
    qr, kr, vr = append_ref(x, heads, kv, hd, positions, g[0], g[1], 1e-6, 1e6)
    for r in range(rows):
        s = int(slots[r])
        if not 0 <= s < n * p:
            assert (out[r] == 7.0).all()
            continue
        close_append(out[r], qr[r], q_t, pairs(qr[r]))
        close_append(k[s // p, s % p], kr[r], kv_t, pairs(kr[r]))
        assert torch.equal(v[s // p, s % p], vr[r].to(kv_t))
        k0[s // p, s % p], v0[s // p, s % p] = k[s // p, s % p], v[s // p, s % p]
    assert torch.equal(k, k0) and torch.equal(v, v0)  # no other slot changed


def test_append_strided_rows_and_new_output():
    torch.manual_seed(2)
    heads, kv, hd, rows = 6, 2, 64, 19
    wide = torch.randn(rows, (heads + 2 * kv) * hd + 64, device="cuda")
    x = wide[:, 64:]
    big = torch.zeros(rows, heads + 3, hd, device="cuda", dtype=BF16)
    k, v = pool(3, 8, kv, hd, BF16, "nhd"), pool(3, 8, kv, hd, BF16, "nhd")
    pos, slots = torch.arange(rows, device="cuda").int(), torch.arange(rows, device="cuda").int()
    paged.paged_append(x, k, v, pos, slots, heads, out=big[:, 1: heads + 1])
    assert (big[:, 0] == 0).all() and (big[:, heads + 1:] == 0).all()
    new = paged.paged_append(x.contiguous(), k, v, pos, slots, heads, q_dtype=BF16)
    assert torch.equal(new, big[:, 1: heads + 1])
    assert paged.paged_append(x[:0], k, v, pos, slots, heads).shape == (0, heads, hd)


# -------------------------------------------------------------- attention

class Case:
    """Requests of given context and new lengths over scattered pages; unused slots and pages hold NaN."""

    def __init__(self, ctx, new, heads, kv, hd, p, q_t, kv_t, layout="nhd", seed=0, spread=1.0, tail_rows=0, spare_cols=2):
        torch.manual_seed(seed)
        self.ctx, self.new, self.heads, self.kv, self.hd, self.p = ctx, new, heads, kv, hd, p
        lens = [c + n for c, n in zip(ctx, new)]
        held = [up(max(n, 0), p) for n in lens]
        n_pages = sum(held) + 3
        order = torch.randperm(n_pages).tolist()
        width = max(max(held), 1) + spare_cols
        self.k, self.v = (pool(n_pages, p, kv, hd, kv_t, layout, float("nan")) for _ in range(2))
        rows, at = [], 0
        for n, h in zip(lens, held):
            pages = order[at: at + h]
            at += h
            rows.append(pages + [order[-1]] * (width - h))
            for i, pg in enumerate(pages):
                m = min(p, n - i * p)
                self.k[pg, :m] = (spread * torch.randn(m, kv, hd, device="cuda")).to(kv_t)
                self.v[pg, :m] = torch.randn(m, kv, hd, device="cuda").to(kv_t)
        self.tables, self.lens = ints(rows), ints(lens)
        self.cu = ints(np.concatenate([[0], np.cumsum(new)]).tolist())
        self.total = sum(new)
        self.q = (spread * torch.randn(self.total + tail_rows, heads, hd, device="cuda")).to(q_t)
        self.scale = 1.0 / math.sqrt(hd)

    def run(self, **kw):
        kw.setdefault("max_new", max(self.new))
        return paged.paged_attention(self.q, self.k, self.v, self.tables, self.cu, self.lens, kw.pop("max_new"), scale=self.scale, **kw)

    def check(self, out, dead=()):
        """Against 64 bits.  Off by at most: the scores' float32 sums (hd roundings and the operands' 2^-24), which move a weight by
        that exponent; the weights' own rounding (bf16: 2^-8, two terms: 2^-16, so do a float32 cache's values), the exponential,
        sums over the keys in float32; the output's rounding to its type."""
        g, qf = self.heads // self.kv, self.q.dtype == F32
        for b, (c, n) in enumerate(zip(self.ctx, self.new)):
            at = int(self.cu[b])
            if n == 0:
                continue
            L = c + n
            pages = self.tables[b].long()
            for h in range(self.kv):
                q = self.q[at: at + n, h * g: (h + 1) * g].double()
                got = out[at: at + n, h * g: (h + 1) * g].double()
                if L <= 0:
                    assert (got == 0).all()
                    continue
                k = self.k[pages[: up(L, self.p)], :, h].double().flatten(0, 1)[:L]
                v = self.v[pages[: up(L, self.p)], :, h].double().flatten(0, 1)[:L]
                pos = torch.arange(c, c + n, device="cuda")
                seen = torch.arange(L, device="cuda") <= pos[:, None]
                for (db, col) in dead:
                    if db == b:
                        seen[:, col * self.p: (col + 1) * self.p] = False
                k, v = k.nan_to_num(0.0), v.nan_to_num(0.0)
                s = torch.einsum("ngd,kd->ngk", q, k) * self.scale
                big = torch.einsum("ngd,kd->ngk", q.abs(), k.abs()) * self.scale
                s = s.masked_fill(~seen[:, None], -math.inf)
                w = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
                tot = w.sum(-1, keepdim=True)
                want = torch.where(tot > 0, torch.einsum("ngk,kd->ngd", w, v) / tot.clamp(min=1e-300), 0.0)
                ds = (big.masked_fill(~seen[:, None], 0).amax(-1, keepdim=True) + 1) * (self.hd + 8) * 2.0 ** -24
                weight = 2.0 ** -8 if not qf else 2.0 ** -16 + (2.0 ** -16 if self.k.dtype == F32 else 0)
                top = v.abs().amax()
                tol = top * (2 * ds + weight + 2.0 ** -21 + L * 2.0 ** -24) + (0 if qf else want.abs() * 2.0 ** -8)
                assert torch.isfinite(got).all()
                assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max().item()


TYPES = [(BF16, BF16), (F32, BF16), (F32, F32)]


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("heads, kv, hd", [(12, 4, 64), (16, 8, 128), (3, 3, 64), (16, 1, 64), (8, 1, 128)])
def test_single_tokens(q_t, kv_t, heads, kv, hd):
    c = Case([0, 1, 7, 15, 16, 17, 62, 63, 64, 65, 127, 128, 300, 1000], [1] * 14, heads, kv, hd, 16, q_t, kv_t, seed=heads)
    c.check(c.run())


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("heads, kv, hd", [(12, 4, 64), (16, 8, 128), (4, 4, 128), (8, 1, 64), (5, 1, 64)])
def test_chunks(q_t, kv_t, heads, kv, hd):
    c = Case([0, 0, 5, 100, 64, 333, 0], [1, 130, 64, 63, 200, 2, 1], heads, kv, hd, 16, q_t, kv_t, seed=hd)
    c.check(c.run())


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("copies", [1, 9, 40])
def test_short_items_beside_long_ones(q_t, kv_t, hd, copies):
    """Items of few rows over one to many key tiles beside items of 256 packed rows, divided and whole, pages missing in some."""
    ctx = [0, 3, 120, 127, 128, 250, 256, 511, 800, 0, 90, 1700] * copies
    new = [6, 1, 8, 1, 64, 65, 20, 1, 63, 140, 128, 2] * copies
    c = Case(ctx, new, 4, 2, hd, 16, q_t, kv_t, seed=18 + copies)
    dead = [(b, col) for b, col in ((2, 7), (5, 0), (7, 8), (8, 3), (11, 40))]
    for b, col in dead:
        c.tables[b, col] = -1
    c.ctx, c.new = ctx[:12] + ctx[-12:], new[:12] + new[-12:]
    out = c.run(max_new=140)
    if copies > 1:  # the first and the last twelve requests
        at = int(c.cu[-13])
        head, n = int(c.cu[12]), int(c.cu[12])
        out = torch.cat([out[:head], out[at:]])
        c.cu = torch.cat([c.cu[:12], c.cu[-13:] - at + n])
        c.tables, c.lens = torch.cat([c.tables[:12], c.tables[-12:]]), torch.cat([c.lens[:12], c.lens[-12:]])
        q = torch.cat([c.q[:head], c.q[at: at + head]])
        c.q = q
    else:
        c.ctx, c.new = ctx, new
    c.check(out, dead)


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("p", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_page_sizes_and_layouts(q_t, kv_t, p, layout):
    one = Case([0, p - 1, p, 3 * p + 1, 500], [1] * 5, 4, 2, 64, p, q_t, kv_t, layout, seed=p)
    one.check(one.run())
    many = Case([0, p, 3 * p + 1, 500, 0], [2 * p + 3, 40, 1, 77, p], 4, 2, 64, p, q_t, kv_t, layout, seed=p + 1)
    many.check(many.run())


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("new", [2, 3, 5, 8, 11, 17])
def test_short_runs(q_t, kv_t, new):
    c = Case([0, 40, 129, 63], [new, 1, new, max(1, new - 1)], 6, 2, 64, 16, q_t, kv_t, seed=new)
    c.check(c.run())


@pytest.mark.parametrize("q_t, kv_t", TYPES)
def test_idle_requests_between_others(q_t, kv_t):
    for new in ([0, 1, 0, 0, 1, 0], [0, 70, 0, 0, 33, 0]):
        c = Case([50, 60, 0, 0, 200, 10], new, 4, 2, 64, 16, q_t, kv_t)
        c.check(c.run())
    none = Case([5, 0], [0, 0], 4, 2, 64, 16, q_t, kv_t, tail_rows=3)
    out = torch.full_like(none.q, 5.0)
    none.run(out=out, max_new=4)
    assert (out == 5.0).all()


@pytest.mark.parametrize("q_t, kv_t", TYPES)
def test_rows_that_see_nothing(q_t, kv_t):
    # fewer tokens than new rows: the first rows sit at negative positions; and no tokens at all
    for new, ctx in (([1, 1, 1], [-1, 3, -1]), ([40, 30, 20], [-7, -30, 4])):
        c = Case(ctx, new, 4, 2, 64, 16, q_t, kv_t, seed=3)
        out = c.run()
        c.check(out)
        for b, (x, n) in enumerate(zip(ctx, new)):
            if x < 0:
                at = int(c.cu[b])
                assert (out[at: at + min(n, -x)] == 0).all()


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("new", [1, 50])
def test_pages_that_do_not_exist_are_hidden(q_t, kv_t, new):
    c = Case([70, 200, 10], [new] * 3, 4, 2, 64, 16, q_t, kv_t, seed=8)
    dead = [(0, 1), (1, 3), (1, 4), (1, 5), (1, 6)]
    for i, (b, col) in enumerate(dead):
        c.tables[b, col] = [-1, c.k.shape[0], 2 ** 31 - 1, -2 ** 31, 10 ** 6][i]
    dead += [(2, i) for i in range(up(10 + new, 16))]
    c.tables[2] = -1  # nothing left to see
    out = c.run()
    saved = c.tables.clone()
    c.tables.clamp_(0, c.k.shape[0] - 1)  # the reference reads some page there and hides it
    c.check(out, dead)
    c.tables.copy_(saved)
    assert (out[int(c.cu[2]):] == 0).all()


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("new", [1, 90])
def test_rows_behind_the_last_request_stay(q_t, kv_t, new):
    c = Case([30, 100], [new, new], 4, 2, 64, 16, q_t, kv_t, tail_rows=9)
    c.q[c.total:] = float("nan")
    out = torch.full_like(c.q, 3.0)
    assert c.run(out=out) is out
    assert (out[c.total:] == 3.0).all()
    c.check(out)


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("new", [1, 40])
def test_strided_queries_and_output(q_t, kv_t, new):
    c = Case([30, 100, 7], [new] * 3, 4, 2, 64, 16, q_t, kv_t)
    wide = torch.zeros(c.total, 9, 64, dtype=q_t, device="cuda")
    wide[:, 2:6] = c.q
    want = c.run()
    c.q = wide[:, 2:6]
    out = torch.zeros(c.total, 7, 64, dtype=q_t, device="cuda")
    c.run(out=out[:, 3:])
    assert torch.equal(out[:, 3:], want) and (out[:, :3] == 0).all()
    c.check(want)


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("new", [1, 30])
def test_large_and_even_scores(q_t, kv_t, new):
    peaked = Case([300, 64], [new] * 2, 4, 2, 64, 16, q_t, kv_t, spread=6.0)
    peaked.check(peaked.run())
    even = Case([300, 64], [new] * 2, 4, 2, 64, 16, q_t, kv_t, spread=0.0)
    even.check(even.run())


@pytest.mark.parametrize("q_t, kv_t", TYPES)
def test_max_new_cuts(q_t, kv_t):
    c = Case([30, 100], [50, 3], 4, 2, 64, 16, q_t, kv_t)
    full = c.run()
    for cut in (1, 20):
        out = torch.full_like(c.q, 9.0)
        c.run(out=out, max_new=cut)
        for b in range(2):
            at, n = int(c.cu[b]), c.new[b]
            done = min(n, cut)
            torch.testing.assert_close(out[at: at + done], full[at: at + done], rtol=2.0 ** -7, atol=2.0 ** -6 * float(full.abs().max()))
            assert (out[at + done: at + n] == 9.0).all()


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_one_long_request_is_divided(q_t, kv_t, hd):
    for new in (1, 20):
        c = Case([20011], [new], 4, 2, hd, 64, q_t, kv_t)
        out = c.run()
        c.check(out)
        assert torch.equal(out, c.run())  # the same call gives the same bits
    c = Case([9000, 3, 0, 12000, 40], [1, 1, 1, 1, 1], 4, 2, hd, 64, q_t, kv_t)
    c.check(c.run())


@pytest.mark.parametrize("q_t, kv_t", TYPES)
def test_many_requests(q_t, kv_t):
    rng = random.Random(4)
    ctx = [rng.choice([0, rng.randint(0, 90)]) for _ in range(1300)]
    for new in ([1] * 1300, [rng.choice([0, 1, 1, 9]) for _ in range(1300)]):
        c = Case(ctx, new, 2, 1, 64, 16, q_t, kv_t)
        c.check(c.run())


def test_offsets_beyond_32_bits():
    """Pools of more than 2^32 bytes and 2^31 elements: the pages at the far end."""
    n, p, kv, hd = 70000, 256, 1, 128
    k = torch.empty(n, p, kv, hd, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    pages = [n - 1, 3, n - 2, 65537]
    for new in (1, 40):
        c = Case([0], [new], 2, kv, hd, p, BF16, BF16)
        L = 3 * p + 100
        ks, vs = torch.randn(L, kv, hd, device="cuda").to(BF16), torch.randn(L, kv, hd, device="cuda").to(BF16)
        for i, pg in enumerate(pages):
            m = min(p, L - i * p)
            k[pg, :m], v[pg, :m] = ks[i * p: i * p + m], vs[i * p: i * p + m]
        c.k, c.v, c.tables, c.ctx, c.lens = k, v, ints([pages]), [L - new], ints([L])
        c.check(c.run())
        x = torch.randn(1, 4 * hd, device="cuda").to(BF16)
        paged.paged_append(x, k, v, ints([5]), ints([(n - 1) * p + 7]), 2)
        assert torch.equal(v[n - 1, 7, 0], x[0, 3 * hd:])


@pytest.mark.parametrize("q_t, kv_t", TYPES)
def test_captured_call_follows_the_lengths(q_t, kv_t):
    big = Case([900, 700, 40], [64, 64, 64], 4, 2, 64, 16, q_t, kv_t, seed=1)
    out = torch.zeros_like(big.q)
    ws = torch.empty(paged.paged_attention_workspace(big.q, big.k, big.v, 64), dtype=torch.uint8, device="cuda")
    big.run(out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        big.run(out=out, workspace=ws)
    for ctx, new in (([900, 700, 40], [64, 64, 64]), ([12, 500, 0], [64, 1, 30]), ([950, 0, 90], [1, 1, 1])):
        big.ctx, big.new = ctx, new
        big.lens.copy_(ints([c + n for c, n in zip(ctx, new)]))
        big.cu.copy_(ints(np.concatenate([[0], np.cumsum(new)]).tolist()))
        graph.replay()
        torch.cuda.synchronize()
        big.check(out)


def test_streams_and_small_workspace():
    c = Case([900, 700, 40], [1, 1, 1], 4, 2, 64, 16, BF16, BF16)
    want = c.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = [c.run(stream=side) for _ in range(3)]
    with torch.cuda.stream(side):
        outs.append(c.run())
    side.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    need = paged.paged_attention_workspace(c.q, c.k, c.v, 1)
    with pytest.raises(CttsError) as e:
        c.run(workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
    assert e.value.code == _lib.ERR_ARG and "workspace" in str(e.value)
    # whatever the workspace held before, and memory behind it is not touched
    ws = torch.full((need + 4096,), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(c.run(workspace=ws), want)
    assert (ws[need:] == 255).all()


# ------------------------------------------------- the three together

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_serving_steps_match_the_contiguous_cache(dtype):
    """One LM layer's attention block over prompts in chunks, decode steps, a release and a new request, through the paged
    operators and ctts_op_linear, against the LM handle with its contiguous cache on the same weights."""
    import ctypes as C

    from helpers import lm_model
    from conftest import cosine, rel_err
    from rcutetts_b200.config import LMConfig
    from rcutetts_b200.model import QwenCache, decode_step, prefill
    from rcutetts_b200 import synth

    cfg = LMConfig(n_layers=1)
    m, w = lm_model(cfg, seed=21, dtype=dtype)
    lib, code = _lib.load(), 1 if dtype == "bf16" else 0

    def dev(a):
        if dtype == "bf16":
            return torch.from_numpy(synth.to_bf16_bits(synth.bf16_round(a)).view(np.int16)).cuda()
        return torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda()

    pre = "layers.0."
    qkv_w = dev(np.concatenate([w[pre + f"self_attn.{n}_proj.weight"] for n in "qkv"]))
    o_w = dev(w[pre + "self_attn.o_proj.weight"])
    gu_w = dev(np.concatenate([w[pre + "mlp.gate_proj.weight"], w[pre + "mlp.up_proj.weight"]]))
    d_w = dev(w[pre + "mlp.down_proj.weight"])
    n1, n2, nf, qn, kn = (torch.from_numpy(np.ascontiguousarray(w[k], np.float32)).cuda() for k in (
        pre + "input_layernorm.weight", pre + "post_attention_layernorm.weight", "norm.weight",
        pre + "self_attn.q_norm.weight", pre + "self_attn.k_norm.weight"))

    def linear(x, wt, n, norm=None, res=None):
        y = torch.empty(x.shape[0], n, device="cuda")
        rc = lib.ctts_op_linear(x.data_ptr(), x.shape[0], x.shape[1], wt.data_ptr(), code, n, 0 if norm is None else norm.data_ptr(),
                                C.c_float(cfg.rms_eps), 0 if res is None else res.data_ptr(), y.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        return y

    H, nq, nkv, hd, F = cfg.hidden, cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, cfg.ffn
    p, batch, n_pages, width = 16, 3, 30, 12
    cache_t = BF16 if dtype == "bf16" else F32
    k, v = (torch.zeros(n_pages, p, nkv, hd, dtype=cache_t, device="cuda") for _ in range(2))
    tables = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(n_pages, device="cuda").int()
    ctx, count = ints([0] * batch), ints([n_pages])
    rng = np.random.default_rng(3)

    def step(rows_of):
        """rows_of[b]: [n, H] new rows, or -1 for a finished request."""
        nonlocal ctx, count
        new = [-1 if isinstance(r, int) else len(r) for r in rows_of]
        x = torch.from_numpy(np.concatenate([r for r in rows_of if not isinstance(r, int)])).cuda()
        s = paged.paged_plan(ctx, ints(new), tables, free, count, p, x.shape[0])
        h = x
        qkv = linear(h, qkv_w, (nq + 2 * nkv) * hd, norm=n1)
        q = paged.paged_append(qkv, k, v, s.positions, s.slots, nq, q_norm=qn, k_norm=kn, eps=cfg.rms_eps, theta=cfg.rope_theta)
        att = paged.paged_attention(q, k, v, tables, s.cu_rows, s.seq_lens, max(max(new), 0))
        h = linear(att.view(-1, nq * hd), o_w, H, res=h)
        gu = linear(h, gu_w, 2 * F, norm=n2)
        act = torch.empty(h.shape[0], F, device="cuda")
        assert lib.ctts_op_swiglu(gu.data_ptr(), h.shape[0], F, act.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        h = linear(act, d_w, H, res=h).double()
        out = (h / torch.sqrt((h ** 2).mean(-1, keepdim=True) + cfg.rms_eps) * nf.double()).cpu().numpy()
        ctx, count = s.seq_lens, s.state
        cu = s.cu_rows.tolist()
        assert s.state[2] == batch
        return [out[cu[b]: cu[b + 1]] for b in range(batch)]

    kvs = [QwenCache(m, batch=1, capacity=192) for _ in range(batch)]

    def contiguous(rows_of):
        out = []
        for b, r in enumerate(rows_of):
            if isinstance(r, int):
                assert lib.ctts_kv_reset(kvs[b].h) == 0
                out.append(np.zeros((0, H), np.float32))
            elif len(r) == 0:
                out.append(np.zeros((0, H), np.float32))
            else:
                out.append(prefill(m, r, kvs[b]) if len(r) > 1 else decode_step(m, r, kvs[b]))
        return out

    def rows(n):
        return rng.standard_normal((n, H), dtype=np.float32)

    steps = [[rows(37), rows(5), rows(0)], [rows(1), rows(40), rows(70)], [rows(1), rows(1), rows(1)], [rows(20), -1, rows(1)],
             [rows(1), rows(33), rows(1)], [rows(1), rows(1), rows(1)]]
    # the gates of the LM's own tests: bf16 weights by direction, float32 by value
    for rows_of in steps:
        for got, want in zip(step(rows_of), contiguous(rows_of)):
            want = np.asarray(want).reshape(-1, H)
            assert got.shape == want.shape
            if want.size:
                assert rel_err(got, want) < 1e-4 if dtype == "f32" else min(cosine(g, x) for g, x in zip(got, want)) >= 0.999


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("new", [1, 3, 40])
def test_other_orders_in_memory(q_t, kv_t, new):
    """Pools as views: keys and values of a page side by side, heads outermost, rows inside wider ones, one page, one head."""
    c = Case([30, 100, 77], [new] * 3, 4, 2, 64, 16, q_t, kv_t, seed=5)
    want = c.run()
    c.check(want)
    n, p, h, d = c.k.shape
    side = torch.stack([c.k, c.v], 1)  # [pages, 2, page, heads, dim]
    heads_out = torch.stack([c.k, c.v]).permute(0, 3, 1, 2, 4).contiguous().permute(0, 2, 3, 1, 4)
    page_in = torch.stack([c.k, c.v]).permute(0, 2, 1, 3, 4).contiguous().permute(0, 2, 1, 3, 4)  # [page slot, pages, ...]
    wide = torch.full((2, n, p, h, d + 8), float("nan"), dtype=kv_t, device="cuda")
    wide[..., 8:] = torch.stack([c.k, c.v])
    for k, v in ((side[:, 0], side[:, 1]), heads_out, page_in, wide[..., 8:]):
        c.k, c.v = k, v
        assert torch.equal(c.run(), want)
    one = Case([5], [new], 2, 1, 64, 256, q_t, kv_t, seed=6, spare_cols=0)
    pg = int(one.tables[0, 0])
    one.k, one.v, one.tables = one.k[pg: pg + 1], one.v[pg: pg + 1], one.tables * 0
    one.check(one.run())


def test_append_other_orders_in_memory():
    torch.manual_seed(9)
    x = torch.randn(20, 8 * 64, device="cuda")
    pos, slots = torch.arange(20, device="cuda").int(), torch.randperm(48, device="cuda")[:20].int()
    k, v = torch.zeros(3, 16, 2, 64, device="cuda"), torch.zeros(3, 16, 2, 64, device="cuda")
    paged.paged_append(x, k, v, pos, slots, 4)
    side, outer = torch.zeros(3, 2, 16, 2, 64, device="cuda"), torch.zeros(2, 2, 3, 16, 64, device="cuda").permute(0, 2, 3, 1, 4)
    for kk, vv in ((side[:, 0], side[:, 1]), outer):
        paged.paged_append(x, kk, vv, pos, slots, 4)
        assert torch.equal(kk, k) and torch.equal(vv, v)


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("ctx, new", [([300, 0, 9000], 1), ([300, 0, 2000], 90)])
def test_output_over_the_queries(q_t, kv_t, ctx, new):
    c = Case(ctx, [new] * 3, 4, 2, 64, 16, q_t, kv_t, seed=12)
    want = c.run()
    c.q = c.q.clone()
    assert torch.equal(c.run(out=c.q), want)


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 70])
def test_bad_values_stay_with_their_request(q_t, kv_t, hd, new):
    """A NaN key, an infinite value or a NaN query reaches the rows that see it and no other request's."""
    c = Case([200, 90, 300], [new] * 3, 4, 2, hd, 16, q_t, kv_t, seed=14)
    want = c.run()
    for j in (0, 3, 6, 7, 130):  # key positions that different parts of a tile hold
        page, slot = int(c.tables[2, j // 16]), j % 16
        keep = c.k[page, slot, 1].clone()
        c.k[page, slot, 1] = float("nan")
        out = c.run()
        c.k[page, slot, 1] = keep
        b2, rest = out[int(c.cu[2]):], out[: int(c.cu[2])]
        assert not torch.isfinite(b2[:, 2:]).any() and torch.equal(b2[:, :2], want[int(c.cu[2]):, :2])
        assert torch.equal(rest, want[: int(c.cu[2])])
    page = int(c.tables[0, 3])
    keep = c.v[page, 5, 0, 7].clone()
    c.v[page, 5, 0, 7] = float("inf")
    out = c.run()
    c.v[page, 5, 0, 7] = keep
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[: new, :2, 7] = True
    assert not torch.isfinite(out[bad]).any() and torch.equal(out[~bad], want[~bad])
    c.q[new // 2, 1, 0] = float("nan")
    out = c.run()
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[new // 2, 1] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], want[~bad])


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
def test_bad_queries_of_short_requests(q_t, kv_t, hd, new):
    """Many short requests, whose items no cut divides: a row whose query is NaN gives NaN, every other what it gave."""
    c = Case([21] * 400, [new] * 400, 4, 2, hd, 16, q_t, kv_t, seed=15)
    want = c.run()
    rows = torch.arange(0, 400, 3, device="cuda") * new + new // 2
    c.q[rows, 3, 5] = float("nan")
    out = c.run()
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[rows, 3] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], want[~bad])


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("scale", [1e-20, 1e20])
def test_scales_at_their_bounds(q_t, kv_t, new, scale):
    """The smallest scale: the mean of the values seen; the largest: the value of the best key."""
    c = Case([37, 300, 2000], [new] * 3, 4, 2, 64, 16, q_t, kv_t, seed=16)
    c.scale = scale
    if scale > 1:  # scores 1 at one key, 0 at the others: weights of exactly 1 and 0
        c.q.zero_()
        c.q[..., 0] = 1.0
        c.k[..., 0] = 0.0
        for b in range(3):
            c.k[int(c.tables[b, 0]), 11, :, 0] = 1.0
    out = c.run().double()
    for b, n in enumerate([37, 300, 2000]):
        v = c.v[c.tables[b].long()].flatten(0, 1).double()[: n + new]  # [tokens, 2, 64]
        for i in range(new):
            want = v[11] if scale > 1 else v[: n + i + 1].mean(0)
            # weights rounded to bf16 are exact here; the sum's float32 adds and one rounding to the output's type
            tol = want.abs() * torch.finfo(q_t).eps / 2 + v[: n + i + 1].abs().mean(0) * (n + i + 1) * 2.0**-23
            assert ((out[b * new + i].view(2, 2, 64) - want[:, None]).abs() <= tol[:, None]).all()


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("sign", [1, -1])
def test_huge_scores(q_t, kv_t, hd, new, sign):
    """Scores of 10^11 and more: the best key takes all, or those within rounding of it share."""
    c = Case([37, 300, 2000] + [21] * 200, [new] * 203, 4, 2, hd, 16, q_t, kv_t, seed=17, spread=1e6)
    c.q, c.k = c.q.abs(), sign * c.k.abs()
    out = c.run().double().view(-1, 2, 2, hd)
    single = 0
    for b in (0, 1, 2, 50, 202):
        L = c.ctx[b] + new
        k, v = (x[c.tables[b].long()].flatten(0, 1)[:L].double() for x in (c.k, c.v))
        for i in range(new):
            s = torch.einsum("hgd,khd->hgk", c.q[b * new + i].view(2, 2, hd).double(), k[: L - new + i + 1])
            # sums of hd terms of one sign, each rounded or cut to 2^-23; the operands' 2^-24 (3 terms)
            close = s >= s.amax(-1, keepdim=True) - s.abs().amax(-1, keepdim=True) * (2 * hd + 4) * 2.0**-23
            got = out[b * new + i]
            for h in range(2):
                for g in range(2):
                    of = v[: L - new + i + 1][close[h, g], h]
                    lo, hi = of.amin(0), of.amax(0)
                    tol = torch.maximum(lo.abs(), hi.abs()) * (2.0**-8 if q_t is BF16 else 2.0**-20)
                    assert ((got[h, g] >= lo - tol) & (got[h, g] <= hi + tol)).all()
                    single += of.shape[0] == 1
    assert single > 0.7 * 5 * new * 4


def test_another_stream_owns_what_it_uses():
    """Calls given a stream: outputs and workspaces come from that stream's memory, so work on the current one cannot reuse them."""
    c = Case([900, 4000, 40], [1, 1, 1], 4, 2, 64, 16, BF16, BF16)
    x = torch.randn(3, 8 * 64, device="cuda").to(BF16)
    want = c.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    need = paged.paged_attention_workspace(c.q, c.k, c.v, 1)
    for how in (side, side.cuda_stream):
        torch.cuda._sleep(2_000_000)  # the current stream is busy
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000)
        outs = []
        for _ in range(4):
            outs.append(c.run(stream=how))
            torch.empty(need, dtype=torch.uint8, device="cuda").fill_(255)
            step = paged.paged_plan(ints([0, 5]), ints([1, 2]), torch.zeros(2, 4, dtype=torch.int32, device="cuda"), ints([1, 2, 3]), ints([3]), 16, 3)
            torch.full((64,), -9, dtype=torch.int32, device="cuda")
        side.synchronize()
        assert all(torch.equal(o, want) for o in outs)
        torch.cuda.synchronize()
        assert step.state.tolist() == [2, 3, 2, 1]
    with pytest.raises((TypeError, AttributeError)):
        c.run(stream="no stream")


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_two_calls_at_once(q_t, kv_t, hd):
    """Chunks and single tokens on two streams at once, and two calls of each kind: every one gives what it gives alone."""
    cases = [Case([900, 0, 300], [200, 70, 1], 4, 2, hd, 16, q_t, kv_t, seed=19), Case([50, 4000, 700], [40, 130, 128], 4, 2, hd, 16, q_t, kv_t, seed=20),
             Case([300, 5000, 12], [1] * 3, 4, 2, hd, 16, q_t, kv_t, seed=21), Case([90] * 70, [1] * 70, 4, 2, hd, 16, q_t, kv_t, seed=22)]
    want = [c.run() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for turn in range(12):
        for k, s in enumerate(streams):
            i = (turn // (3 * k + 1) + k) % 4
            with torch.cuda.stream(s):
                got.append((i, cases[i].run()))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i]) for i, out in got)


def test_captured_runs_on_two_streams():
    """Two captured steps with workspaces of their own, replayed at once."""
    cases = [Case([900, 0, 300], [200, 70, 1], 4, 2, 128, 16, BF16, BF16, seed=23), Case([50, 4000], [1, 1], 4, 2, 64, 16, F32, BF16, seed=24)]
    want = [c.run() for c in cases]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in cases], [], []
    for c, s in zip(cases, streams):
        out = torch.empty_like(c.q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for _ in range(3):
                c.run(out=out)
        graphs.append(g)
        outs.append(out)
    for _ in range(5):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
