"""How exact attention with float32 queries is: every operand carries 24 bits.

The inputs make a score one product (a query and a key share one dimension
that is not zero) and an output value one weight times one value (the value of
key j is zero but in dimension j), so that few roundings lie on the way and the
bound is far below what losing the last 8 bits of any operand costs."""
import math

import pytest
import torch

from test_paged_gpu import BF16, F32, Case

L = 12  # keys of a request


def bound(S, terms):
    """Relative error of an output w_j v_j / sum for scores up to S, in units of 2^-23; `terms` products a pair of operands (6, or 3
    over a bf16 cache).

    Score: the products that are left out (second times third term, both ways) 1; each of `terms` added, the sum cut to 2^-23 of
    itself, and one addition of the small ones to the leading one: terms + 1, of |s| <= S.
    Argument: difference, factor and product, 2^-24 each, of up to 2 S: 3 S.  (The maximum's own error shifts all weights alike.)
    Exponential: 2 (two units in the last place).  Merge of partial states: an argument, an exponential and a product more: 3 S + 3.
    Output: both the weight and the sum of the weights have that error, the sum L additions of 2^-24; the weight's and value's rest
    behind three terms 2^-24 each, left out products 1, `terms` additions cut, four merged states 2, reciprocal and product 1."""
    weight = (terms + 2) * S + 3 * S + 2 + 3 * S + 3
    return (2 * weight + L / 2 + 1 + 1 + terms + 2 + 1) * 2.0**-23


def inputs(heads, kv, hd, new, kv_t, S, seed, n=40):
    """n requests of L tokens: a Case, factors of the queries a [rows, heads], of the keys b [n, L, kv], values c [n, L, kv]."""
    g = torch.Generator().manual_seed(seed)

    def mantissas(*shape):
        return (1 + torch.rand(*shape, generator=g)) * (2 * torch.randint(0, 2, shape, generator=g) - 1)

    a, b, c = mantissas(n * new, heads), mantissas(n, L, kv).to(kv_t).float(), mantissas(n, L, kv).to(kv_t).float()
    return a, b, c, S / 4  # |a b| < 4


def outputs(a, b, c, scale, heads, kv, new, terms=None, cut=None):
    """[n * new, heads, L] in 64 bits; `cut`: the operand that keeps only its first `terms` bf16 terms."""

    def of(name, x):
        if name != cut:
            return x
        kept = torch.zeros_like(x)
        for _ in range(terms):
            kept = kept + (x - kept).float().to(BF16).double()
        return kept

    n, group = b.shape[0], heads // kv
    q = of("q", a.double()).view(n, new, kv, group)
    s = torch.einsum("nihg,njh->nihgj", q, of("k", b.double())) * scale
    seen = torch.arange(L) <= (L - new + torch.arange(new))[:, None]
    s = s.masked_fill(~seen[None, :, None, None], -math.inf)
    w = torch.exp(s - s.amax(-1, keepdim=True))
    out = of("w", w) * of("v", c.double()).permute(0, 2, 1)[:, None, :, None] / w.sum(-1, keepdim=True)
    return out.reshape(n * new, heads, L)


SHAPES = [(12, 4, 64, 1), (16, 8, 128, 1), (16, 1, 64, 1), (16, 1, 128, 1), (12, 4, 64, 4), (16, 8, 128, 7), (12, 4, 64, 6), (16, 1, 128, 8),
          (12, 4, 128, 12), (4, 4, 64, 12)]


@pytest.mark.parametrize("kv_t", [F32, BF16])
@pytest.mark.parametrize("S", [4.0, 1 / 16])
def test_bound_is_below_a_missing_term(kv_t, S):
    """What the test below could not see it would not be worth: two terms of one operand break the bound, scores' at large ones."""
    a, b, c, scale = inputs(4, 4, 64, 6, kv_t, S, 1)
    want = outputs(a, b, c, scale, 4, 4, 6)
    tol = bound(S, 6 if kv_t == F32 else 3) * want.abs()
    for cut in (("q", "k") if S > 1 else ("w", "v")):
        got = outputs(a, b, c, scale, 4, 4, 6, terms=2, cut=cut)
        seen = bool(((got - want).abs() > tol).any())
        assert seen == (kv_t == F32 or cut in "qw"), cut  # (a bf16 cache has one term)
        whole = outputs(a, b, c, scale, 4, 4, 6, terms=3, cut=cut)
        assert ((whole - want).abs() <= tol / 16).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kv_t", [F32, BF16])
@pytest.mark.parametrize("S", [4.0, 1 / 16])
@pytest.mark.parametrize("heads, kv, hd, new", SHAPES)
def test_float32_queries_carry_24_bits(heads, kv, hd, new, kv_t, S):
    a, b, c, scale = inputs(heads, kv, hd, new, kv_t, S, heads + hd + new)
    n = b.shape[0]
    case = Case([L - new] * n, [new] * n, heads, kv, hd, 8, F32, kv_t)
    case.q.zero_()
    heads_of = torch.arange(heads)
    case.q[:, heads_of, (7 * (heads_of // (heads // kv)) + 3) % hd] = a.cuda()
    case.scale = scale
    for r in range(n):
        for j in range(L):
            page, slot = int(case.tables[r, j // 8]), j % 8
            case.k[page, slot], case.v[page, slot] = 0, 0
            case.k[page, slot, torch.arange(kv), (7 * torch.arange(kv) + 3) % hd] = b[r, j].to(kv_t).cuda()
            case.v[page, slot, :, j] = c[r, j].to(kv_t).cuda()
    out = case.run().double().cpu()
    want = outputs(a, b, c, scale, heads, kv, new)
    assert (out[..., L:] == 0).all()
    assert ((out[..., :L] - want).abs() <= bound(S, 6 if kv_t == F32 else 3) * want.abs()).all()
