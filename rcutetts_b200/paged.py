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
import functools
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


def _bad_ints(what, dev):
    raise ValueError(f"{what} must be contiguous int32 tensors on one CUDA device" + ("" if dev >= 0 else " (the paged operators run on CUDA tensors)"))


def _run(fn, dev: int, args: bytes, stream):
    """The call on device `dev`, on its current stream or the given one."""
    if dev < 0:
        raise ValueError("the paged operators run on CUDA tensors")
    if stream is None:
        stream = torch._C._cuda_getCurrentRawStream(dev)  # torch.cuda.current_stream without making a Stream object
    elif not isinstance(stream, int):
        stream = stream.cuda_stream
    if dev == torch._C._cuda_getDevice():
        rc = fn(args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(args, stream)
    if rc:
        check(rc)


def _pool(k: torch.Tensor, v: torch.Tensor):
    """The C ABI's ctts_paged_kv of a pair of pools."""
    shape, stride, dtype = k.shape, k.stride(), _TYPES.get(k.dtype)
    if len(shape) != 4 or v.shape != shape or v.stride() != stride or v.dtype is not k.dtype or v.get_device() != k.get_device():
        raise ValueError("the pools are two [pages, page_size, kv heads, head dim] tensors of one type and layout on one device")
    if dtype is None:
        raise ValueError("a cache is float32 or bf16")
    n, p, h, d = shape
    sp, st, sh, sd = stride
    if sd != 1:
        raise ValueError("the head dim of a pool is contiguous")
    # the stride of a dimension of one carries no meaning: one that passes the checks
    return (k.data_ptr(), v.data_ptr(), sp if n > 1 else p * h * d, st, sh if h > 1 else d, n, p, h, d, dtype)


def _table(block_tables, batch, dev):
    """Row stride and width of the block tables."""
    shape = block_tables.shape
    if block_tables.dtype is not torch.int32 or block_tables.get_device() != dev or len(shape) != 2 or shape[0] != batch:
        raise ValueError("block_tables must be an int32 [batch, pages] tensor on the other tensors' device")
    ld, col = block_tables.stride()
    if col != 1 and shape[1] > 1:
        raise ValueError("a row of block_tables is contiguous")
    return (ld if batch > 1 else max(ld, shape[1])), shape[1]


def paged_plan(ctx_lens, new_lens, block_tables, free_pages, free_count, page_size: int, max_rows: int, stream=None) -> PagedStep:
    """Block tables, row offsets, positions and slots of a step from the request lengths.

    ctx_lens, new_lens [batch] (new > 0: rows, 0: idle, < 0: finished), block_tables [batch, max_pages] (updated in place: pages
    taken), free_pages (a stack, updated in place: pages given back), free_count [1 or more] (its first entry counts), all int32
    on one device.
    """
    dev, batch = ctx_lens.get_device(), ctx_lens.numel()
    for t in (ctx_lens, new_lens, free_pages, free_count):
        if t.dtype is not torch.int32 or t.get_device() != dev or not t.is_contiguous():
            _bad_ints("ctx_lens, new_lens, free_pages and free_count", dev)
    if new_lens.numel() != batch or free_count.numel() < 1:
        raise ValueError("ctx_lens and new_lens have one entry per request, free_count at least one")
    ld, pages = _table(block_tables, batch, dev)
    if max_rows < 0:
        raise ValueError("max_rows must not be negative")
    # one allocation: lengths, offsets, state, positions, slots
    out = ctx_lens.new_empty(2 * batch + 5 + 2 * max_rows)
    at = out.data_ptr()
    cu = at + 4 * batch
    state = cu + 4 * batch + 4
    pos = state + 16
    _run(_lib.load().ctts_op_paged_plan, dev,
         _PLAN.pack(ctx_lens.data_ptr(), new_lens.data_ptr(), free_count.data_ptr(), block_tables.data_ptr(), free_pages.data_ptr(),
                    at, cu, pos, pos + 4 * max_rows, state, ld, batch, page_size, pages, free_pages.numel(), max_rows), stream)
    a, b, c, d, e = out.split_with_sizes([batch, batch + 1, 4, max_rows, max_rows])
    return PagedStep(a, b, d, e, c)


def paged_append(x, k_pages, v_pages, positions, slots, n_heads: int, q_norm=None, k_norm=None, eps: float = 1e-6, theta: float = 1e6,
                 q_dtype: Optional[torch.dtype] = None, out=None, stream=None):
    """QK-Norm and RoPE of the rows x [rows, (n_heads + 2 kv heads) * head dim]; keys and values go to their slots of the pools,
    the queries [rows, n_heads, head dim] are returned (in `out`, whose rows without a slot are left as they were, or a new tensor
    of q_dtype, x's type unless given, whose rows without a slot are undefined)."""
    dev, kv = x.get_device(), _pool(k_pages, v_pages)
    hd, shape, x_t = kv[8], x.shape, _TYPES.get(x.dtype)
    if len(shape) != 2 or x_t is None or shape[1] != (n_heads + 2 * kv[7]) * hd or k_pages.get_device() != dev:
        raise ValueError("x must be a float32 or bf16 [rows, (n_heads + 2 * kv heads) * head dim] tensor on the pools' device")
    rows = shape[0]
    x_ld, x_col = x.stride()
    if x_col != 1:
        raise ValueError("a row of x is contiguous")
    for t in (positions, slots):
        if t.dtype is not torch.int32 or t.get_device() != dev or not t.is_contiguous() or t.numel() < rows:
            _bad_ints("positions and slots (one entry per row)", dev)
    gains = [0, 0]
    for i, g in enumerate((q_norm, k_norm)):
        if g is not None:
            if g.dtype is not torch.float32 or g.get_device() != dev or not g.is_contiguous() or g.numel() != hd:
                raise ValueError("q_norm and k_norm are float32 [head dim] tensors")
            gains[i] = g.data_ptr()
    if out is None:
        out = x.new_empty((rows, n_heads, hd), dtype=q_dtype or x.dtype)
    elif out.shape != (rows, n_heads, hd) or out.get_device() != dev or (q_dtype is not None and out.dtype is not q_dtype):
        raise ValueError("out must be a float32 or bf16 [rows, n_heads, head dim] tensor on x's device")
    q_t = _TYPES.get(out.dtype)
    q_ld, q_h, q_d = out.stride()
    if q_t is None or q_d != 1 or (n_heads > 1 and q_h != hd):
        raise ValueError("queries are float32 or bf16, a row of them is contiguous")
    if rows < 2:
        x_ld, q_ld = shape[1], n_heads * hd
    _run(_lib.load().ctts_op_paged_append, dev,
         _APPEND.pack(*kv, x.data_ptr(), out.data_ptr(), positions.data_ptr(), slots.data_ptr(), gains[0], gains[1], x_ld, q_ld, theta, eps,
                      rows, n_heads, x_t, q_t), stream)
    return out


def paged_attention(q, k_pages, v_pages, block_tables, cu_rows, seq_lens, max_new: int, scale: Optional[float] = None, out=None,
                    workspace=None, stream=None):
    """Causal attention of the rows q [rows, heads, head dim] over the pages of their requests; max_new bounds a request's rows.

    Returns [rows, heads, head dim] in q's type (`out`, whose rows behind the last request are left as they were, or a new tensor).
    workspace: a uint8 tensor of paged_attention_workspace bytes to use instead of one from torch's allocator.
    """
    dev, kv = q.get_device(), _pool(k_pages, v_pages)
    hd, shape, dtype, q_t = kv[8], q.shape, q.dtype, _TYPES.get(q.dtype)
    if len(shape) != 3 or shape[2] != hd or q_t is None or k_pages.get_device() != dev:
        raise ValueError("q must be a float32 or bf16 [rows, heads, head dim] tensor on the pools' device")
    rows, heads, _ = shape
    q_ld, q_h, q_d = q.stride()
    if q_d != 1 or (heads > 1 and q_h != hd):
        raise ValueError("a row of q is contiguous")
    for t in (cu_rows, seq_lens):
        if t.dtype is not torch.int32 or t.get_device() != dev or not t.is_contiguous():
            _bad_ints("cu_rows and seq_lens", dev)
    batch = seq_lens.numel()
    if cu_rows.numel() != batch + 1:
        raise ValueError("cu_rows has one entry more than seq_lens")
    t_ld, pages = _table(block_tables, batch, dev)
    width = heads * hd
    if out is None:
        out = torch.empty_like(q) if q_ld == width else q.new_empty(shape)
        o_ld = width
    else:
        if out.shape != shape or out.dtype is not dtype or out.get_device() != dev:
            raise ValueError("out must have q's shape and type, on its device")
        o_ld, o_h, o_d = out.stride()
        if o_d != 1 or (heads > 1 and o_h != hd):
            raise ValueError("a row of out is contiguous")
    if rows < 2:
        q_ld = o_ld = width
    need = _workspace_bytes(dev, kv[5:], heads, max_new, q_t)
    if workspace is None:
        workspace = q.new_empty(need, dtype=torch.uint8)
        have = need
    else:
        if workspace.get_device() != dev or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous tensor on q's device")
        have = workspace.numel() * workspace.element_size()
    _run(_lib.load().ctts_op_paged_attention, dev,
         _ATTN.pack(*kv, q.data_ptr(), out.data_ptr(), block_tables.data_ptr(), cu_rows.data_ptr(), seq_lens.data_ptr(), workspace.data_ptr(),
                    have, q_ld, o_ld, t_ld, batch, rows, heads, pages, max_new, q_t, 1.0 / math.sqrt(hd) if scale is None else scale), stream)
    return out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(dev: int, pool, heads: int, max_new: int, q_t: int) -> int:
    """Workspace of a call: it follows from the device, the pools' sizes and type, the heads, the rows' bound and the queries' type."""
    if dev < 0:
        raise ValueError("the paged operators run on CUDA tensors")
    need, hd = C.c_size_t(), pool[3]
    args = _ATTN.pack(0, 0, hd, hd, hd, *pool, 0, 0, 0, 0, 0, 0, 0, heads * hd, heads * hd, 1, 1, 1, heads, 1, max_new, q_t, 1.0)
    with torch.cuda.device(dev):
        check(_lib.load().ctts_op_paged_attention_workspace(args, C.byref(need)))
    return need.value


def paged_attention_workspace(q, k_pages, v_pages, max_new: int) -> int:
    """Bytes of a workspace that serves calls on these tensors with up to max_new new rows a request."""
    return _workspace_bytes(q.get_device(), _pool(k_pages, v_pages)[5:], q.shape[1], max_new, _TYPES[q.dtype])
