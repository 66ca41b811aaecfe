"""The paged KV-cache operators: what is measured, and their plain forms.

One serving step over a paged cache is a run of three operators:

  plan       request lengths -> block tables, page grants and releases, row
             offsets, positions and slots of the step's new rows
  append     QK-Norm and RoPE of the new rows, keys and values into their slots
  attention  the new rows of every request over its pages, causal

A case is a dict of plain values.  With `own` false, `run` is elementary torch
arithmetic in 32 bits (angles in 64); with `own` true it calls the framework.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one decode step's book-keeping for the benchmark's 64 utterances
        dict(name="plan_decode_b64", op="plan", batch=64, page=16, ctx_lo=120, ctx_hi=1200, new_lo=1, new_hi=1, single=1.0,
             idle=0.0, done=0.0, pad=0, mix=1),
        # a large scheduler step: chunked prefills beside decodes, idle and finished requests
        dict(name="plan_mixed_b1500", op="plan", batch=1500, page=16, ctx_lo=1, ctx_hi=8000, new_lo=2, new_hi=512, single=0.6,
             idle=0.1, done=0.1, pad=77, mix=2),
        # the new rows of one decode step, bf16 weights (float32 activations, bf16 cache)
        dict(name="append_decode_b64", op="append", rows=64, pad=0, n_heads=12, n_kv=4, hd=64, page=16, x="f32", q="f32", kv="bf16",
             layout="nhd", far=1200, mix=3),
        # a long prompt of the shipped model, everything in bf16
        dict(name="append_chunk_bf16", op="append", rows=16381, pad=3, n_heads=16, n_kv=8, hd=128, page=64, x="bf16", q="bf16",
             kv="bf16", layout="hnd", far=60000, mix=4),
        # a prompt of the float32 model
        dict(name="append_chunk_f32", op="append", rows=4001, pad=0, n_heads=12, n_kv=4, hd=64, page=32, x="f32", q="f32", kv="f32",
             layout="nhd", far=9000, mix=5),
        # one utterance, one token, float32 throughout: latency
        dict(name="decode_b1_f32", op="attention", batch=1, ctx_lo=300, ctx_hi=300, new_lo=1, new_hi=1, single=1.0, n_heads=12,
             n_kv=4, hd=64, page=16, q="f32", kv="f32", layout="nhd", mix=6),
        # the batched decode step of the benchmark: 64 utterances of mixed age
        dict(name="decode_b64", op="attention", batch=64, ctx_lo=150, ctx_hi=1200, new_lo=1, new_hi=1, single=1.0, n_heads=12,
             n_kv=4, hd=64, page=16, q="f32", kv="bf16", layout="nhd", mix=7),
        # long ragged contexts of the shipped model's heads: the cache does not fit L2
        dict(name="decode_long_bf16", op="attention", batch=30, ctx_lo=2000, ctx_hi=32000, new_lo=1, new_hi=1, single=1.0, n_heads=16,
             n_kv=8, hd=128, page=64, q="bf16", kv="bf16", layout="hnd", mix=8),
        # chunks of long prompts after an existing context: the largest
        dict(name="chunk_bf16", op="attention", batch=4, ctx_lo=4000, ctx_hi=6100, new_lo=1500, new_hi=2048, single=0.0, n_heads=16,
             n_kv=8, hd=128, page=64, q="bf16", kv="bf16", layout="nhd", mix=9),
        # whole prompts at once, bf16 cache under float32 activations
        dict(name="prompt_f32q", op="attention", batch=8, ctx_lo=0, ctx_hi=0, new_lo=190, new_hi=900, single=0.0, n_heads=12,
             n_kv=4, hd=64, page=16, q="f32", kv="bf16", layout="nhd", mix=10),
        # chunks in float32 throughout
        dict(name="chunk_f32", op="attention", batch=2, ctx_lo=100, ctx_hi=1000, new_lo=700, new_hi=1500, single=0.0, n_heads=12,
             n_kv=4, hd=64, page=32, q="f32", kv="f32", layout="hnd", mix=11),
        # a serving step: decodes and a few prompt chunks in one call
        dict(name="mixed_bf16", op="attention", batch=48, ctx_lo=100, ctx_hi=2000, new_lo=200, new_hi=512, single=0.9, n_heads=12,
             n_kv=4, hd=64, page=16, q="bf16", kv="bf16", layout="nhd", mix=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(max(hi, 1))))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attention", "attention", "attention"])
    mix = rng.randrange(1, 1 << 30)
    page = rng.choice([8, 16, 16, 32, 64, 128, 256])
    if op == "plan":
        batch = _log(rng, 1, 2000)
        return dict(op=op, batch=batch, page=page, ctx_lo=rng.choice([0, 1, 50]), ctx_hi=_log(rng, 60, 8000), new_lo=1,
                    new_hi=_log(rng, 1, 512), single=rng.choice([0.0, 0.5, 0.9]), idle=rng.choice([0.0, 0.2]),
                    done=rng.choice([0.0, 0.1, 0.4]), pad=rng.choice([0, 1, 130]), mix=mix)
    x, kv = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "bf16")])
    n_kv = rng.choice([1, 2, 4, 8])
    n_heads = n_kv * rng.choice([1, 2, 3, 4, 8] if n_kv < 8 else [1, 2, 3])
    hd = rng.choice([64, 128])
    layout = rng.choice(["nhd", "hnd"])
    if op == "append":
        rows = _log(rng, 1, 16000 * 32 * 128 // ((n_heads + 2 * n_kv) * hd) if x == "bf16" else 8000 * 32 * 128 // ((n_heads + 2 * n_kv) * hd))
        return dict(op=op, rows=min(rows, 30000), pad=rng.choice([0, 5]), n_heads=n_heads, n_kv=n_kv, hd=hd, page=page, x=x, q=x, kv=kv,
                    layout=layout, far=_log(rng, 64, 100000), mix=mix)
    single = rng.choice([0.0, 0.0, 0.8, 1.0, 1.0])
    batch, top = (_log(rng, 1, 100), 32000) if single == 1.0 else (_log(rng, 1, 40 if single else 12), 6000)
    ctx_hi = _log(rng, 1, top)
    ctx_lo = rng.choice([0, ctx_hi // 10, ctx_hi])
    new_hi = 1 if single == 1.0 else _log(rng, 2, 2048)
    new_lo = max(1, new_hi // rng.choice([1, 3, 50]))
    while batch > 1 and (batch * new_hi * (ctx_hi + new_hi) * n_heads > 9e8 or batch * (ctx_hi + new_hi) * n_kv * hd > 7e8):
        batch -= 1
    while new_hi * (ctx_hi + new_hi) * n_heads > 9e8:
        ctx_hi = ctx_hi // 2
        ctx_lo = min(ctx_lo, ctx_hi)
    return dict(op=op, batch=batch, ctx_lo=ctx_lo, ctx_hi=ctx_hi, new_lo=new_lo, new_hi=new_hi, single=single, n_heads=n_heads, n_kv=n_kv,
                hd=hd, page=page, q=x, kv=kv, layout=layout, mix=mix)


def _lengths(case):
    """Context and new rows of every request: they follow from the case, the values from the seed."""
    rng = random.Random(case["mix"])
    n = case["batch"]
    ctx = [_log(rng, case["ctx_lo"], case["ctx_hi"]) for _ in range(n)]
    new = [1 if rng.random() < case["single"] else _log(rng, case["new_lo"], case["new_hi"]) for _ in range(n)]
    if case["op"] == "plan":
        for b in range(n):
            u = rng.random()
            if u < case["idle"]:
                new[b] = 0
            elif u < case["idle"] + case["done"]:
                new[b] = -1
    return ctx, new


def _up(n, d):
    return -(-n // d)


# ----------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + case["mix"])
    return {"plan": _prepare_plan, "append": _prepare_append, "attention": _prepare_attention}[case["op"]](case, gen)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _pool(case, gen, n_pages):
    """A pool [pages, page, kv heads, head dim] of values with some head-wise scale, in the case's memory layout."""
    p, h, d = case["page"], case["n_kv"], case["hd"]
    if case["layout"] == "hnd":
        return _randn(gen, n_pages, h, p, d).to(TYPES[case["kv"]]).transpose(1, 2)
    return _randn(gen, n_pages, p, h, d).to(TYPES[case["kv"]])


def _tables(held, width, order):
    """Rows of `order`'s pages, held[b] of them for request b; the rest of a row is -1."""
    held = held.long()
    first = held.cumsum(0) - held
    col = torch.arange(width, device="cuda")
    at = (first[:, None] + col).clamp(max=order.numel() - 1)
    return torch.where(col < held[:, None], order[at], -1).to(torch.int32)


def _prepare_plan(case, gen):
    ctx, new = _lengths(case)
    p = case["page"]
    held = sum(_up(c, p) for c in ctx)
    need = sum(_up(c + n, p) - _up(c, p) for c, n in zip(ctx, new) if n > 0)
    n_pages = held + need + 9  # the step fits, with a few pages to spare
    width = max(_up(c + max(n, 0), p) for c, n in zip(ctx, new)) + 2
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    tables = _tables(_ints([_up(c, p) for c in ctx]), width, order[: max(held, 1)])
    free = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
    free[: n_pages - held] = order[held:]
    return dict(op="plan", page=p, ctx=_ints(ctx), new=_ints(new), tables=tables, free=free, count=_ints([n_pages - held]),
                max_rows=sum(n for n in new if n > 0) + case["pad"])


def _prepare_append(case, gen):
    rows, pad, p, far = case["rows"], case["pad"], case["page"], case["far"]
    n_pages = _up(rows, p) + 5
    width = (case["n_heads"] + 2 * case["n_kv"]) * case["hd"]
    x = _randn(gen, rows + pad, width).to(TYPES[case["x"]])
    slots = torch.randperm(n_pages * p, generator=gen, device="cuda")[: rows + pad].to(torch.int32)
    slots[rows:] = -1
    positions = torch.randint(0, far, (rows + pad,), generator=gen, device="cuda", dtype=torch.int32)
    positions[rows:] = -1
    k, v = _pool(case, gen, n_pages), _pool(case, gen, n_pages)
    gains = 1.0 + 0.3 * _randn(gen, 2, case["hd"])
    out = torch.zeros(rows + pad, case["n_heads"], case["hd"], dtype=TYPES[case["q"]], device="cuda")
    return dict(op="append", rows=rows, heads=case["n_heads"], x=x, slots=slots, positions=positions, k=k, v=v, q_norm=gains[0].contiguous(),
                k_norm=gains[1].contiguous(), eps=1e-6, theta=1e6, out=out)


def _prepare_attention(case, gen):
    ctx, new = _lengths(case)
    p = case["page"]
    lens = [c + n for c, n in zip(ctx, new)]
    held = [_up(n, p) for n in lens]
    n_pages = sum(held) + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    # queries and keys after QK-Norm: their products have a standard deviation of about two
    q = (1.5 * _randn(gen, cu[-1], case["n_heads"], case["hd"])).to(TYPES[case["q"]])
    k, v = _pool(case, gen, n_pages), _pool(case, gen, n_pages)
    if case["kv"] == "f32" or n_pages * p * case["n_kv"] * case["hd"] < 1 << 28:
        k.mul_(1.4)
    return dict(op="attention", q=q, k=k, v=v, tables=_tables(_ints(held), max(held) + 1, order), cu=_ints(cu), lens=_ints(lens),
                max_new=max(new), max_len=max(lens), scale=1.0 / math.sqrt(case["hd"]))


# -------------------------------------------------------------- the passes

def run(s):
    if own:
        from rcutetts_b200 import paged

        if s["op"] == "plan":
            step = paged.paged_plan(s["ctx"], s["new"], s["tables"], s["free"], s["count"], s["page"], s["max_rows"])
            return {"tables": s["tables"], "free": s["free"], "lens": step.seq_lens, "cu": step.cu_rows, "positions": step.positions,
                    "slots": step.slots, "state": step.state}
        if s["op"] == "append":
            q = paged.paged_append(s["x"], s["k"], s["v"], s["positions"], s["slots"], s["heads"], q_norm=s["q_norm"],
                                   k_norm=s["k_norm"], eps=s["eps"], theta=s["theta"], out=s["out"])
            return {"q": q, "k": s["k"], "v": s["v"]}
        return {"out": paged.paged_attention(s["q"], s["k"], s["v"], s["tables"], s["cu"], s["lens"], s["max_new"], scale=s["scale"])}
    return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention}[s["op"]](s)


def _plain_plan(s):
    """Finished requests (new < 0) give their pages back, on top of the free stack in request and page order.  The others are
    granted in order, each new page from the top of the stack, up to the first that does not fit (pages, table width, rows)."""
    ctx, new, p = s["ctx"].long(), s["new"].long(), s["page"]
    tables, free = s["tables"], s["free"]
    count = s["count"][0].long()
    col = torch.arange(tables.shape[1], device=ctx.device)
    held = (ctx + p - 1) // p
    done = new < 0
    gone = torch.where(done, held, 0)
    gone_first = gone.cumsum(0) - gone
    stack = torch.cat([free, free.new_zeros(1)])
    to = torch.where(col < gone[:, None], count + gone_first[:, None] + col, free.numel())
    stack.scatter_(0, to.flatten(), tables.flatten())
    free.copy_(stack[:-1])
    avail = count + gone.sum()

    rows = new.clamp(min=0)
    after = torch.where(rows > 0, (ctx + rows + p - 1) // p, held)
    need = torch.where(done, 0, after - held)
    fits = (need.cumsum(0) <= avail) & (rows.cumsum(0) <= s["max_rows"]) & ((after <= tables.shape[1]) | (rows == 0))
    granted = fits.long().cumprod(0)
    rows, need = rows * granted, need * granted
    first = need.cumsum(0) - need
    j = col - held[:, None]
    fresh = (j >= 0) & (j < need[:, None])
    at = (avail - 1 - first[:, None] - j).clamp(min=0, max=free.numel() - 1)
    tables.copy_(torch.where(fresh, free[at], tables))

    ends = rows.cumsum(0)
    cu = torch.cat([ends.new_zeros(1), ends])
    r = torch.arange(s["max_rows"], device=ctx.device)
    b = torch.searchsorted(ends, r, right=True).clamp(max=ctx.numel() - 1)
    real = r < ends[-1]
    pos = torch.where(real, ctx[b] + r - cu[b], 0)
    slots = torch.where(real, tables[b, pos // p].long() * p + pos % p, -1)
    taken = need.sum()
    state = torch.stack([avail - taken, ends[-1], granted.sum(), taken])
    return {"tables": tables, "free": free, "lens": torch.where(done, 0, ctx + rows).int(), "cu": cu.int(),
            "positions": torch.where(real, pos, -1).int(), "slots": slots.int(), "state": state.int()}


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_append(s):
    rows, heads, k, v = s["rows"], s["heads"], s["k"], s["v"]
    kv, hd, p = k.shape[2], k.shape[3], k.shape[1]
    x = s["x"][:rows].float().view(rows, heads + 2 * kv, hd)
    freq = s["theta"] ** (-torch.arange(0, hd, 2, device=x.device, dtype=torch.float64) / hd)
    angle = s["positions"][:rows, None].double() * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    qk = x[:, : heads + kv]
    qk = qk * (qk.square().mean(-1, keepdim=True) + s["eps"]).rsqrt()
    s["out"][:rows] = _rotate(qk[:, :heads] * s["q_norm"], cos, sin).to(s["out"].dtype)
    slot = s["slots"][:rows].long()
    k[slot // p, slot % p] = _rotate(qk[:, heads:] * s["k_norm"], cos, sin).to(k.dtype)
    v[slot // p, slot % p] = x[:, heads + kv:].to(v.dtype)
    return {"q": s["out"], "k": k, "v": v}


def _plain_attention(s):
    """Softmax over the keys 0..position of each row, computed on a padded batch."""
    q, k, v = s["q"], s["k"], s["v"]
    p, kv, hd = k.shape[1:]
    heads, n = q.shape[1], s["max_new"]
    pages = _up(s["max_len"], p)
    tables = s["tables"][:, :pages].clamp(min=0).long()
    batch = tables.shape[0]
    cu, lens = s["cu"].long(), s["lens"].long()
    i = torch.arange(n, device=q.device)
    count = cu[1:] - cu[:-1]
    row = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qs = q[row].float().view(batch, n, kv, heads // kv, hd).permute(0, 2, 3, 1, 4).reshape(batch, kv, -1, hd)
    ks = k[tables].float().reshape(batch, pages * p, kv, hd).permute(0, 2, 3, 1)
    score = torch.matmul(qs, ks)
    del ks
    score = score.mul_(s["scale"]).view(batch, kv, heads // kv, n, pages * p)
    pos = (lens - count)[:, None] + i
    hidden = torch.arange(pages * p, device=q.device) > pos[:, :, None]
    score.masked_fill_(hidden[:, None, None], -math.inf)
    weight = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = weight.sum(-1, keepdim=True)
    vs = v[tables].float().reshape(batch, pages * p, kv, hd).permute(0, 2, 1, 3)
    out = torch.matmul(weight.view(batch, kv, -1, pages * p), vs).view(batch, kv, heads // kv, n, hd) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(batch * n, heads, hd).to(q.dtype)
    at = torch.arange(q.shape[0], device=q.device)
    b = torch.searchsorted(cu[1:], at, right=True)
    return {"out": out[b * n + at - cu[b]]}


# ------------------------------------------------------- what it has to do

def work(case):
    op = case["op"]
    if op == "plan":
        ctx, new = _lengths(case)
        p, batch = case["page"], case["batch"]
        rows = sum(n for n in new if n > 0)
        taken = sum(_up(c + n, p) - _up(c, p) for c, n in zip(ctx, new) if n > 0)
        gone = sum(_up(c, p) for c, n in zip(ctx, new) if n < 0)
        # lengths in; lengths and offsets out; pages moved from one list to another; position and slot of each row; the pages begun before
        return {"bytes": 4 * (2 * batch + 2 * batch + 1 + 2 * taken + 2 * gone + 2 * (rows + case["pad"]) + batch + 5), "flops": 4 * (rows + batch)}
    size = {"f32": 4, "bf16": 2}
    hd, heads, kv = case["hd"], case["n_heads"], case["n_kv"]
    if op == "append":
        rows = case["rows"]
        moved = size[case["x"]] * (heads + 2 * kv) + size[case["q"]] * heads + size[case["kv"]] * 2 * kv
        return {"bytes": rows * (hd * moved + 8) + 8 * hd, "flops": rows * hd * (heads + kv) * 7}
    ctx, new = _lengths(case)
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, new))
    keys = sum(c + n for c, n in zip(ctx, new))
    tables = sum(_up(c + n, case["page"]) for c, n in zip(ctx, new))
    return {"bytes": 2 * size[case["q"]] * sum(new) * heads * hd + 2 * size[case["kv"]] * keys * kv * hd + 4 * (tables + 2 * len(ctx)),
            "flops": 4 * pairs * heads * hd}


# ------------------------------------------------------- in 64 bits, apart

def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers: they have to be equal
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attention(s, case)


def _exact_append(s):
    kv, hd, p = s["k"].shape[2], s["k"].shape[3], s["k"].shape[1]
    heads, rows = s["heads"], s["rows"]
    x = s["x"][:rows].double().unflatten(1, (heads + 2 * kv, hd))
    turn = torch.pow(torch.tensor(s["theta"], dtype=torch.float64, device=x.device), torch.arange(hd // 2, device=x.device).double() * (-2.0 / hd))
    # a pair (d, d + hd/2) is a complex number, and a position turns it
    unit = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), s["positions"][:rows].double()[:, None, None] * turn)

    def turned(y, gain):
        y = y / torch.sqrt(torch.linalg.vector_norm(y, dim=-1, keepdim=True) ** 2 / hd + s["eps"]) * gain.double()
        z = torch.complex(y[..., : hd // 2], y[..., hd // 2:]) * unit
        return torch.cat([z.real, z.imag], -1)

    q = s["out"].double()
    q[:rows] = turned(x[:, :heads], s["q_norm"])
    k, v = s["k"].double(), s["v"].double()
    page, off = torch.div(s["slots"][:rows].long(), p, rounding_mode="floor"), s["slots"][:rows].long() % p
    k.index_put_((page, off), turned(x[:, heads: heads + kv], s["k_norm"]))
    v.index_put_((page, off), x[:, heads + kv:])
    return {"q": q, "k": k, "v": v}


def _exact_attention(s, case):
    """Request by request and KV head by KV head."""
    ctx, new = _lengths(case)
    q, p = s["q"], case["page"]
    group = case["n_heads"] // case["n_kv"]
    out, at = torch.zeros(q.shape, dtype=torch.float64, device=q.device), 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        pages = s["tables"][b, : _up(c + n, p)].long()
        seen = torch.tril(torch.ones(n, c + n, dtype=torch.bool, device=q.device), diagonal=c)
        for h in range(case["n_kv"]):
            k = s["k"][pages, :, h].double().flatten(0, 1)[: c + n]
            v = s["v"][pages, :, h].double().flatten(0, 1)[: c + n]
            mine = q[at: at + n, h * group: (h + 1) * group].double()
            score = torch.einsum("ngd,kd->gnk", mine, k) * s["scale"]
            share = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
            out[at: at + n, h * group: (h + 1) * group] = torch.einsum("gnk,kd->ngd", share, v)
        at += n
    return {"out": out}
