"""Paged KV-cache operators on torch CUDA tensors.

One serving step over a paged cache is a run of three calls:

    step = paged_plan(ctx_lens, new_lens, block_tables, free_pages, free_count, page_size, max_rows)
    q = paged_append(qkv, k_pages, v_pages, step.positions, step.slots, n_heads, q_norm=..., k_norm=...)
    out = paged_attention(q, k_pages, v_pages, block_tables, step.cu_rows, step.seq_lens, max_new)

(the contracts are those of ctts_op_paged_plan / _append / _attention in
include/cutetts_b200.h).  The pools k_pages and v_pages are [pages, page_size,
kv heads, head dim] tensors of float32 or bf16 with any order in memory; one
pair per layer.  For inference: no gradients flow through the calls (what they
write in place counts as a new version of its tensor).  They run on the tensors'
device, on its current stream unless `stream` is given, and can be captured in a
CUDA graph.  Arguments of a wrong type, shape or device raise ValueError, what
the library refuses CttsError: a step without requests, for one.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib

_lib.load()  # the library the binding is linked to
try:
    from . import _paged_ext as _ext
except ImportError as e:
    raise ImportError(f"{e}: build the binding with `python -m rcutetts_b200.build`") from e

_ext.set_error(_lib.CttsError)

_TYPES = {None: -1, torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}


class PagedStep(NamedTuple):
    """What paged_plan says about the step (all int32, on the device)."""

    seq_lens: torch.Tensor   # [batch] lengths with the step's rows; the next step's ctx_lens
    cu_rows: torch.Tensor    # [batch + 1] row offsets
    positions: torch.Tensor  # [max_rows], -1 behind the last row
    slots: torch.Tensor      # [max_rows], -1 behind the last row
    state: torch.Tensor      # [4] free pages now (the next step's free_count), rows, requests ahead of the first refused one, pages taken


def paged_plan(ctx_lens, new_lens, block_tables, free_pages, free_count, page_size: int, max_rows: int, stream=None) -> PagedStep:
    """Block tables, row offsets, positions and slots of a step from the request lengths.

    ctx_lens, new_lens [batch] (new > 0: rows, 0: idle, < 0: finished), block_tables [batch, max_pages] (updated in place: pages
    taken), free_pages (a stack, updated in place: pages given back), free_count [1 or more] (its first entry counts), all int32
    on one device.
    """
    return PagedStep._make(_ext.plan(ctx_lens, new_lens, block_tables, free_pages, free_count, page_size, max_rows, stream))


def paged_append(x, k_pages, v_pages, positions, slots, n_heads: int, q_norm=None, k_norm=None, eps: float = 1e-6, theta: float = 1e6,
                 q_dtype: Optional[torch.dtype] = None, out=None, stream=None) -> torch.Tensor:
    """QK-Norm and RoPE of the rows x [rows, (n_heads + 2 kv heads) * head dim]; keys and values go to their slots of the pools,
    the queries [rows, n_heads, head dim] are returned (in `out`, whose rows without a slot are left as they were, or a new tensor
    of q_dtype, x's type unless given, whose rows without a slot are undefined)."""
    if q_dtype not in _TYPES:
        raise ValueError("queries are float32 or bf16")
    return _ext.append(x, k_pages, v_pages, positions, slots, n_heads, q_norm, k_norm, eps, theta, _TYPES[q_dtype], out, stream)


def paged_attention(q, k_pages, v_pages, block_tables, cu_rows, seq_lens, max_new: int, scale: Optional[float] = None, out=None,
                    workspace=None, stream=None) -> torch.Tensor:
    """Causal attention of the rows q [rows, heads, head dim] over the pages of their requests; max_new bounds a request's rows
    (pass the step's own bound: a generous one costs time, see ctts_op_paged_attention).

    Returns [rows, heads, head dim] in q's type (`out`, whose rows behind the last request are left as they were, or a new tensor).
    workspace: a tensor of paged_attention_workspace bytes or more to use instead of one from torch's allocator; calls that may
    overlap need one each.
    """
    return _ext.attention(q, k_pages, v_pages, block_tables, cu_rows, seq_lens, max_new, scale, out, workspace, stream)


def paged_attention_workspace(q, k_pages, v_pages, max_new: int) -> int:
    """Bytes of a workspace that serves calls on these tensors with up to max_new new rows a request."""
    return _ext.attention_workspace(q, k_pages, v_pages, max_new)
