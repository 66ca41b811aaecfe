"""Promises of the paged KV-cache operators beyond their formulas: a workspace
sized once serves every shorter call."""
import pytest
import torch

from rcutetts_b200 import paged
from test_paged_gpu import BF16, F32, TYPES, Case

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
