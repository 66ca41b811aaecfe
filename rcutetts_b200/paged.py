"""Paged KV-cache operators on torch CUDA tensors.

One serving step over a paged cache is a run of three calls:

    step = paged_plan(ctx_lens, new_lens, block_tables, free_pages, free_count, page_size, max_rows)
    q = paged_append(qkv, k_pages, v_pages, step.positions, step.slots, n_heads, q_norm=..., k_norm=...)
    out = paged_attention(q, k_pages, v_pages, block_tables, step.cu_rows, step.seq_lens, max_new)

(the contracts are those of ctts_op_paged_plan / _append / _attention in
include/cutetts_b200.h).  The pools k_pages and v_pages are [pages, page_size,
kv heads, head dim] tensors of float32 or bf16 with any order in memory; one
pair per layer.  Calls run on the tensors' device, on its current stream
unless `stream` is given, and can be captured in a CUDA graph.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import check

_TYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16}

# the argument structs of the C ABI, packed in one go (native order and alignment)
_KV = "PPqqqiiiii4x"
_PLAN = struct.Struct("@PPPPPPPPPPqiiiii4x")
_APPEND = struct.Struct("@" + _KV + "PPPPPPqqdfiiii4x")
_ATTN = struct.Struct("@" + _KV + "PPPPPPNqqqiiiiiif4x")


class PagedStep(NamedTuple):
    """What paged_plan says about the step (all int32, on the device)."""

    seq_lens: torch.Tensor   # [batch] lengths with the step's rows; the next step's ctx_lens
    cu_rows: torch.Tensor    # [batch + 1] row offsets
    positions: torch.Tensor  # [max_rows], -1 behind the last row
    slots: torch.Tensor      # [max_rows], -1 behind the last row
    state: torch.Tensor      # [4] free pages now (the next step's free_count), rows, requests ahead of the first refused one, pages taken


def _ints(device, **named):
    for name, t in named.items():
        if t.dtype != torch.int32 or t.device != device or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor on {device}")


def _run(fn, device, args: bytes, stream):
    """The call on the tensors' device, on its current stream or the given one."""
    if device.type != "cuda":
        raise ValueError("the paged operators run on CUDA tensors")
    if stream is None:
        stream = torch.cuda.current_stream(device).cuda_stream
    elif not isinstance(stream, int):
        stream = stream.cuda_stream
    if device.index == torch.cuda.current_device():
        check(fn(args, stream))
    else:
        with torch.cuda.device(device):
            check(fn(args, stream))


def _pool(k: torch.Tensor, v: torch.Tensor):
    """The C ABI's ctts_paged_kv of a pair of pools."""
    if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device:
        raise ValueError("the pools are two [pages, page_size, kv heads, head dim] tensors of one type and layout")
    if k.dtype not in _TYPES:
        raise ValueError("a cache is float32 or bf16")
    n, p, h, d = k.shape
    sp, st, sh, sd = k.stride()
    if sd != 1:
        raise ValueError("the head dim of a pool is contiguous")
    # the stride of a dimension of one carries no meaning: one that passes the checks
    return (k.data_ptr(), v.data_ptr(), sp if n > 1 else p * h * d, st, sh if h > 1 else d, n, p, h, d, _TYPES[k.dtype])


def paged_plan(ctx_lens, new_lens, block_tables, free_pages, free_count, page_size: int, max_rows: int, stream=None) -> PagedStep:
    """Block tables, row offsets, positions and slots of a step from the request lengths.

    ctx_lens, new_lens [batch] (new > 0: rows, 0: idle, < 0: finished), block_tables [batch, max_pages] (updated in place: pages
    taken), free_pages (a stack, updated in place: pages given back), free_count [1 or more] (its first entry counts), all int32
    on one device.
    """
    device = ctx_lens.device
    _ints(device, ctx_lens=ctx_lens, new_lens=new_lens, free_pages=free_pages, free_count=free_count)
    batch = ctx_lens.numel()
    if new_lens.numel() != batch or free_count.numel() < 1:
        raise ValueError("ctx_lens and new_lens have one entry per request, free_count at least one")
    if (block_tables.dtype != torch.int32 or block_tables.device != device or block_tables.dim() != 2 or
            block_tables.shape[0] != batch or (block_tables.shape[1] > 1 and block_tables.stride(1) != 1)):
        raise ValueError(f"block_tables must be an int32 [batch, pages] tensor on {device}")
    if max_rows < 0:
        raise ValueError("max_rows must not be negative")
    # one allocation: lengths, offsets, state, positions, slots
    out = torch.empty(2 * batch + 5 + 2 * max_rows, dtype=torch.int32, device=device)
    at = out.data_ptr()
    lens, cu, state, pos, slots = (at, at + 4 * batch, at + 4 * (2 * batch + 1), at + 4 * (2 * batch + 5), at + 4 * (2 * batch + 5 + max_rows))
    pages = block_tables.shape[1]
    _run(_lib.load().ctts_op_paged_plan, device,
         _PLAN.pack(ctx_lens.data_ptr(), new_lens.data_ptr(), free_count.data_ptr(), block_tables.data_ptr(), free_pages.data_ptr(),
                    lens, cu, pos, slots, state, max(block_tables.stride(0), pages) if batch == 1 else block_tables.stride(0), batch,
                    page_size, pages, free_pages.numel(), max_rows), stream)
    a, b, c, d, e = out.split_with_sizes([batch, batch + 1, 4, max_rows, max_rows])
    return PagedStep(a, b, d, e, c)


def paged_append(x, k_pages, v_pages, positions, slots, n_heads: int, q_norm=None, k_norm=None, eps: float = 1e-6, theta: float = 1e6,
                 q_dtype: Optional[torch.dtype] = None, out=None, stream=None):
    """QK-Norm and RoPE of the rows x [rows, (n_heads + 2 kv heads) * head dim]; keys and values go to their slots of the pools,
    the queries [rows, n_heads, head dim] are returned (in `out`, whose rows without a slot are left as they were, or a new tensor
    of q_dtype, x's type unless given, whose rows without a slot are undefined)."""
    device = x.device
    kv = _pool(k_pages, v_pages)
    rows, hd = x.shape[0], kv[8]
    if x.dim() != 2 or x.shape[1] != (n_heads + 2 * kv[7]) * hd or x.stride(1) != 1 or x.dtype not in _TYPES or k_pages.device != device:
        raise ValueError("x must be a float32 or bf16 [rows, (n_heads + 2 * kv heads) * head dim] tensor on the pools' device")
    _ints(device, positions=positions, slots=slots)
    if positions.numel() < rows or slots.numel() < rows:
        raise ValueError("positions and slots have one entry per row")
    for g in (q_norm, k_norm):
        if g is not None and (g.dtype != torch.float32 or g.numel() != hd or not g.is_contiguous() or g.device != device):
            raise ValueError("q_norm and k_norm are float32 [head dim] tensors")
    if out is None:
        out = torch.empty((rows, n_heads, hd), dtype=q_dtype or x.dtype, device=device)
    elif out.shape != (rows, n_heads, hd) or out.device != device or out.dtype not in _TYPES or out.stride(2) != 1 or (n_heads > 1 and out.stride(1) != hd):
        raise ValueError("out must be a float32 or bf16 [rows, n_heads, head dim] tensor with whole rows")
    if out.dtype not in _TYPES:
        raise ValueError("queries are float32 or bf16")
    width = n_heads * hd
    _run(_lib.load().ctts_op_paged_append, device,
         _APPEND.pack(*kv, x.data_ptr(), out.data_ptr(), positions.data_ptr(), slots.data_ptr(),
                      0 if q_norm is None else q_norm.data_ptr(), 0 if k_norm is None else k_norm.data_ptr(),
                      x.stride(0) if rows > 1 else x.shape[1], out.stride(0) if rows > 1 else width, theta, eps, rows, n_heads,
                      _TYPES[x.dtype], _TYPES[out.dtype]), stream)
    return out


def paged_attention(q, k_pages, v_pages, block_tables, cu_rows, seq_lens, max_new: int, scale: Optional[float] = None, out=None,
                    workspace=None, stream=None):
    """Causal attention of the rows q [rows, heads, head dim] over the pages of their requests; max_new bounds a request's rows.

    Returns [rows, heads, head dim] in q's type (`out`, whose rows behind the last request are left as they were, or a new tensor).
    workspace: a uint8 tensor of paged_attention_workspace bytes to use instead of one from torch's allocator.
    """
    device = q.device
    kv = _pool(k_pages, v_pages)
    hd = kv[8]
    if q.dim() != 3 or q.shape[2] != hd or q.dtype not in _TYPES or k_pages.device != device:
        raise ValueError("q must be a float32 or bf16 [rows, heads, head dim] tensor on the pools' device")
    rows, heads, _ = q.shape
    sq, sh, sd = q.stride()
    if sd != 1 or (heads > 1 and sh != hd):
        raise ValueError("a row of q is contiguous")
    _ints(device, cu_rows=cu_rows, seq_lens=seq_lens)
    batch = seq_lens.numel()
    if cu_rows.numel() != batch + 1:
        raise ValueError("cu_rows has one entry more than seq_lens")
    if (block_tables.dtype != torch.int32 or block_tables.device != device or block_tables.dim() != 2 or
            block_tables.shape[0] != batch or (block_tables.shape[1] > 1 and block_tables.stride(1) != 1)):
        raise ValueError(f"block_tables must be an int32 [batch, pages] tensor on {device}")
    if out is None:
        out = torch.empty((rows, heads, hd), dtype=q.dtype, device=device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != device or out.stride(2) != 1 or (heads > 1 and out.stride(1) != hd):
        raise ValueError("out must have q's shape and type, and whole rows")
    width, pages = heads * hd, block_tables.shape[1]
    tail = (sq if rows > 1 else width, out.stride(0) if rows > 1 else width,
            max(block_tables.stride(0), pages) if batch == 1 else block_tables.stride(0), batch, rows, heads, pages, max_new,
            _TYPES[q.dtype], 1.0 / math.sqrt(hd) if scale is None else scale)
    lib = _lib.load()
    if workspace is None:
        workspace = torch.empty(_workspace_bytes(lib, device, kv, tail), dtype=torch.uint8, device=device)
    elif workspace.device != device or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous tensor on q's device")
    _run(lib.ctts_op_paged_attention, device,
         _ATTN.pack(*kv, q.data_ptr(), out.data_ptr(), block_tables.data_ptr(), cu_rows.data_ptr(), seq_lens.data_ptr(),
                    workspace.data_ptr(), workspace.numel() * workspace.element_size(), *tail), stream)
    return out


def _workspace_bytes(lib, device, kv, tail) -> int:
    need = C.c_size_t()
    args = _ATTN.pack(*kv, 0, 0, 0, 0, 0, 0, 0, *tail)
    if device.type != "cuda":
        raise ValueError("the paged operators run on CUDA tensors")
    with torch.cuda.device(device):
        check(lib.ctts_op_paged_attention_workspace(args, C.byref(need)))
    return need.value


def paged_attention_workspace(q, k_pages, v_pages, max_new: int) -> int:
    """Bytes of a workspace that serves calls on these tensors with up to max_new new rows a request."""
    rows, heads, hd = q.shape
    kv = _pool(k_pages, v_pages)
    return _workspace_bytes(_lib.load(), q.device, kv, (heads * hd, heads * hd, 1, 1, rows, heads, 1, max_new, _TYPES[q.dtype], 1.0))
