"""Promises of the paged KV-cache operators beyond their formulas: a workspace
sized once serves every shorter call, and torch sees what is written in place."""
import pytest
import torch

from rcutetts_b200 import paged
from test_paged_gpu import BF16, F32, TYPES, Case, ints, pool

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------- workspaces

def workspaces(q_t, kv_t, group, hd, most):
    q = torch.empty(1, group, hd, dtype=q_t, device="cuda")
    k = torch.empty(1, 16, 1, hd, dtype=kv_t, device="cuda")
    return [paged.paged_attention_workspace(q, k, k, n) for n in range(1, most + 1)]


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_workspace_grows_with_the_new_rows(q_t, kv_t, hd):
    for group in range(1, 17):
        need = workspaces(q_t, kv_t, group, hd, 40)
        assert need == sorted(need), (group, need)


@pytest.mark.parametrize("q_t, kv_t", TYPES)
@pytest.mark.parametrize("heads, kv, hd, most", [(12, 4, 64, 5), (16, 8, 128, 3), (16, 8, 128, 8), (8, 1, 128, 2), (3, 3, 64, 14), (2, 2, 128, 40)])
def test_workspace_of_short_runs_serves_single_tokens(q_t, kv_t, heads, kv, hd, most):
    for new in range(1, most + 1):
        c = Case([300, 0, 2000], [new] * 3, heads, kv, hd, 16, q_t, kv_t, seed=new)
        ws = torch.empty(paged.paged_attention_workspace(c.q, c.k, c.v, most), dtype=torch.uint8, device="cuda")
        c.check(c.run(workspace=ws))


# ------------------------------------------------------ writes in place

def test_writes_in_place_count_as_versions():
    """torch tells by a tensor's version whether something it has saved was changed since."""
    tables, free, count = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), ints([1, 2, 3]), ints([3])
    ctx, new = ints([0, 5]), ints([1, 2])
    read, written = (ctx, new, count), (tables, free)
    before = [t._version for t in read + written]
    step = paged.paged_plan(ctx, new, tables, free, count, 16, 3)
    assert [t._version for t in read] == before[:3] and all(t._version > v for t, v in zip(written, before[3:]))

    x = torch.randn(3, 8 * 64, device="cuda")
    k, v = pool(5, 16, 2, 64, F32, "nhd"), pool(5, 16, 2, 64, F32, "nhd")
    out = torch.empty(3, 4, 64, device="cuda")
    before = [t._version for t in (x, step.slots, k, v, out)]
    paged.paged_append(x, k, v, step.positions, step.slots, 4, out=out)
    assert [t._version for t in (x, step.slots)] == before[:2] and all(t._version > b for t, b in zip((k, v, out), before[2:]))

    q = out.clone()
    before = [t._version for t in (q, k, v, tables, out)]
    paged.paged_attention(q, k, v, tables, step.cu_rows, step.seq_lens, 2, out=out)
    assert [t._version for t in (q, k, v, tables)] == before[:4] and out._version > before[4]
    view = out[:, 1:]  # a view shares its base's version
    paged.paged_attention(q[:, 1:].clone()[:, :2], k, v, tables, step.cu_rows, step.seq_lens, 2, out=view[:, :2])
    assert out._version > before[4] + 1


def test_a_saved_tensor_that_was_overwritten_is_noticed():
    k, v = pool(5, 16, 2, 64, F32, "nhd"), pool(5, 16, 2, 64, F32, "nhd")
    w = torch.randn_like(k).requires_grad_()
    loss = (w * k).sum()  # saves the pool for w's gradient
    paged.paged_append(torch.randn(1, 8 * 64, device="cuda"), k, v, ints([0]), ints([7]), 4)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors():
    """They have no versions; the calls take them all the same."""
    with torch.inference_mode():
        c = Case([30, 100], [1, 1], 4, 2, 64, 16, BF16, BF16)
        out = torch.empty_like(c.q)
        c.check(c.run(out=out))
        x = torch.randn(2, 8 * 64, device="cuda")
        k, v = pool(5, 16, 2, 64, F32, "nhd"), pool(5, 16, 2, 64, F32, "nhd")
        paged.paged_append(x, k, v, ints([0, 1]), ints([7, 8]), 4)
        assert torch.equal(v[0, 7:9].flatten(1), x[:, 6 * 64:])
        assert paged.paged_plan(ints([0]), ints([1]), ints([[0]]), ints([3]), ints([1]), 16, 1).slots.tolist() == [48]
