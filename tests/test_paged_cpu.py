"""Refusals of the paged KV-cache operators that need no GPU: every argument
the host can see is checked before anything is launched."""
import ctypes as C
import os
import struct

import pytest
import torch

from rcutetts_b200 import _lib, build

if not (os.path.exists(_lib.LIB_PATH) and os.path.exists(build.EXT)):
    build.build()
from rcutetts_b200 import paged  # noqa: E402

# the argument structs of the C ABI (native order and alignment)
POOL = "PPqqqiiiii4x"
STRUCT = {"plan": struct.Struct("@PPPPPPPPPPqiiiii4x"), "append": struct.Struct("@" + POOL + "PPPPPPqqdfiiii4x"),
          "attention": struct.Struct("@" + POOL + "PPPPPPNqqqiiiiiif4x")}
PTR = 1 << 20  # a 16-byte aligned address that is never looked at


def call(name, args):
    lib = _lib.load()
    rc = getattr(lib, name)(args, None)
    return rc, lib.ctts_last_error().decode()


KV = dict(k=PTR, v=PTR, ps=16 * 4 * 64, ts=4 * 64, hs=64, n=10, p=16, h=4, d=64, t=1)
PLAN = dict(ctx=PTR, new=PTR + 64, count=PTR + 128, tables=PTR + 256, free=PTR + 512, lens=PTR + 1024, cu=PTR + 2048, pos=PTR + 4096,
            slots=PTR + 8192, state=PTR + 16384, ld=8, batch=4, p=16, pages=8, cap=10, rows=20)
APPEND = dict(KV, x=PTR, q=PTR, pos=PTR, slots=PTR, qn=PTR, kn=PTR, xld=20 * 64, qld=12 * 64, theta=1e6, eps=1e-6, rows=3, heads=12, xt=0, qt=0)
ATTN = dict(KV, q=PTR, out=PTR, tables=PTR, cu=PTR, lens=PTR, ws=PTR, wsb=1 << 40, qld=12 * 64, old=12 * 64, tld=8, batch=2, rows=5, heads=12,
            pages=8, new=4, qt=0, scale=0.125)


def pack(kind, **over):
    d = dict({"plan": PLAN, "append": APPEND, "attention": ATTN}[kind], **over)
    return STRUCT[kind].pack(*d.values())


@pytest.mark.parametrize("kind", ["plan", "append", "attention"])
def test_null_struct(kind):
    rc, msg = call(f"ctts_op_paged_{kind}", None)
    assert rc == _lib.ERR_ARG and "null" in msg


@pytest.mark.parametrize("over, code", [
    (dict(ctx=0), _lib.ERR_ARG), (dict(new=0), _lib.ERR_ARG), (dict(count=0), _lib.ERR_ARG), (dict(tables=0), _lib.ERR_ARG),
    (dict(free=0), _lib.ERR_ARG), (dict(lens=0), _lib.ERR_ARG), (dict(cu=0), _lib.ERR_ARG), (dict(pos=0), _lib.ERR_ARG),
    (dict(slots=0), _lib.ERR_ARG), (dict(state=0), _lib.ERR_ARG), (dict(batch=0), _lib.ERR_ARG), (dict(batch=-1), _lib.ERR_ARG),
    (dict(batch=4097), _lib.ERR_RANGE), (dict(p=12), _lib.ERR_ARG), (dict(p=4), _lib.ERR_ARG), (dict(p=512), _lib.ERR_ARG),
    (dict(p=0), _lib.ERR_ARG), (dict(pages=0), _lib.ERR_ARG), (dict(ld=7), _lib.ERR_ARG), (dict(rows=-1), _lib.ERR_ARG),
    (dict(cap=-1), _lib.ERR_ARG), (dict(pages=1 << 28, ld=1 << 28), _lib.ERR_RANGE),
    # outputs on inputs: the lengths, and the free count inside the state
    (dict(lens=PTR), _lib.ERR_ARG), (dict(lens=PTR + 12), _lib.ERR_ARG), (dict(state=PTR + 128), _lib.ERR_ARG),
    (dict(state=PTR + 116), _lib.ERR_ARG), (dict(cu=PTR + 64), _lib.ERR_ARG), (dict(pos=PTR), _lib.ERR_ARG), (dict(slots=PTR - 4), _lib.ERR_ARG),
])
def test_plan_refuses(over, code):
    assert call("ctts_op_paged_plan", pack("plan", **over))[0] == code


POOL_BAD = [
    (dict(d=96), _lib.ERR_ARG), (dict(d=256), _lib.ERR_ARG), (dict(t=2), _lib.ERR_ARG), (dict(n=0), _lib.ERR_ARG), (dict(h=0), _lib.ERR_ARG),
    (dict(p=24), _lib.ERR_ARG), (dict(p=4), _lib.ERR_ARG), (dict(p=512), _lib.ERR_ARG), (dict(n=1 << 28), _lib.ERR_RANGE),
    (dict(ps=1), _lib.ERR_ARG), (dict(ts=65), _lib.ERR_ARG), (dict(hs=60), _lib.ERR_ARG), (dict(ts=-64), _lib.ERR_ARG),
    (dict(k=0), _lib.ERR_ARG), (dict(v=0), _lib.ERR_ARG), (dict(k=PTR + 8), _lib.ERR_ARG), (dict(v=PTR + 2), _lib.ERR_ARG),
]


@pytest.mark.parametrize("over, code", POOL_BAD + [
    (dict(x=0), _lib.ERR_ARG), (dict(q=0), _lib.ERR_ARG), (dict(pos=0), _lib.ERR_ARG), (dict(slots=0), _lib.ERR_ARG), (dict(qn=0), _lib.ERR_ARG),
    (dict(kn=0), _lib.ERR_ARG), (dict(xld=19 * 64), _lib.ERR_ARG), (dict(xld=20 * 64 + 1), _lib.ERR_ARG), (dict(qld=11 * 64), _lib.ERR_ARG),
    (dict(theta=0.0), _lib.ERR_ARG), (dict(theta=float("nan")), _lib.ERR_ARG), (dict(theta=float("inf")), _lib.ERR_ARG), (dict(eps=-1.0), _lib.ERR_ARG),
    (dict(eps=float("nan")), _lib.ERR_ARG), (dict(rows=-1), _lib.ERR_ARG), (dict(heads=10), _lib.ERR_ARG), (dict(heads=0), _lib.ERR_ARG),
    (dict(xt=2), _lib.ERR_ARG), (dict(qt=-1), _lib.ERR_ARG), (dict(x=PTR + 4), _lib.ERR_ARG), (dict(q=PTR + 8), _lib.ERR_ARG),
    (dict(qn=PTR + 4), _lib.ERR_ARG), (dict(kn=PTR + 8), _lib.ERR_ARG), (dict(rows=0x7fffffff), _lib.ERR_RANGE),
])
def test_append_refuses(over, code):
    assert call("ctts_op_paged_append", pack("append", **over))[0] == code


@pytest.mark.parametrize("over, code", POOL_BAD + [
    (dict(q=0), _lib.ERR_ARG), (dict(out=0), _lib.ERR_ARG), (dict(tables=0), _lib.ERR_ARG), (dict(cu=0), _lib.ERR_ARG), (dict(lens=0), _lib.ERR_ARG),
    (dict(ws=0), _lib.ERR_ARG), (dict(heads=10), _lib.ERR_ARG), (dict(heads=68, qld=68 * 64, old=68 * 64), _lib.ERR_ARG),
    (dict(qt=2), _lib.ERR_ARG), (dict(qt=1, t=0), _lib.ERR_ARG), (dict(batch=0), _lib.ERR_ARG), (dict(rows=-1), _lib.ERR_ARG),
    (dict(new=-1), _lib.ERR_ARG), (dict(pages=0), _lib.ERR_ARG), (dict(tld=7), _lib.ERR_ARG), (dict(qld=11 * 64), _lib.ERR_ARG),
    (dict(old=12 * 64 + 2), _lib.ERR_ARG), (dict(scale=0.0), _lib.ERR_ARG), (dict(scale=-1.0), _lib.ERR_ARG), (dict(scale=float("nan")), _lib.ERR_ARG),
    (dict(scale=float("inf")), _lib.ERR_ARG), (dict(q=PTR + 8), _lib.ERR_ARG), (dict(out=PTR + 4), _lib.ERR_ARG), (dict(ws=PTR + 4), _lib.ERR_ARG),
    (dict(pages=1 << 28, tld=1 << 28), _lib.ERR_RANGE), (dict(rows=0x7fffffff), _lib.ERR_RANGE),
])
def test_attention_refuses(over, code):
    assert call("ctts_op_paged_attention", pack("attention", **over))[0] == code


@pytest.mark.parametrize("scale", [1e-21, 1e-45, 2e20, 3e38])
def test_attention_refuses_a_scale_whose_factor_vanishes_or_overflows(scale):
    assert call("ctts_op_paged_attention", pack("attention", scale=scale))[0] == _lib.ERR_ARG


def test_attention_refuses_keys_and_heads_past_32_bits():
    over = dict(pages=1 << 26, tld=1 << 26, h=64, heads=64, qld=64 * 64, old=64 * 64)
    assert call("ctts_op_paged_attention", pack("attention", **over))[0] == _lib.ERR_RANGE
    over.update(rows=0, h=32, heads=32, qld=32 * 64, old=32 * 64)  # half as many fit
    assert call("ctts_op_paged_attention", pack("attention", **over))[0] == 0


def test_nothing_to_do_is_no_error():
    assert call("ctts_op_paged_append", pack("append", rows=0))[0] == 0
    assert call("ctts_op_paged_attention", pack("attention", rows=0))[0] == 0
    assert call("ctts_op_paged_attention", pack("attention", new=0))[0] == 0


def test_workspace_refuses():
    lib, need = _lib.load(), C.c_size_t()
    assert lib.ctts_op_paged_attention_workspace(None, C.byref(need)) == _lib.ERR_ARG
    assert lib.ctts_op_paged_attention_workspace(pack("attention"), None) == _lib.ERR_ARG
    assert lib.ctts_op_paged_attention_workspace(pack("attention", heads=10), C.byref(need)) == _lib.ERR_ARG


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_python_checks():
    pool = torch.zeros(4, 16, 2, 64)
    x, q = torch.zeros(3, 8 * 64), torch.zeros(3, 4, 64)
    with pytest.raises(ValueError):  # no CUDA tensors
        paged.paged_plan(_i(2), _i(2), _i(2, 3), _i(4), _i(1), 16, 5)
    with pytest.raises(ValueError):
        paged.paged_plan(_i(2).long(), _i(2), _i(2, 3), _i(4), _i(1), 16, 5)
    with pytest.raises(ValueError):
        paged.paged_plan(_i(2), _i(3), _i(2, 3), _i(4), _i(1), 16, 5)
    with pytest.raises(ValueError):
        paged.paged_plan(_i(2), _i(2), _i(3, 2).t(), _i(4), _i(1), 16, 5)
    with pytest.raises(ValueError):
        paged.paged_plan(_i(2), _i(2), _i(2, 3), _i(4), _i(1), 16, -1)
    with pytest.raises(ValueError):
        paged.paged_append(x, pool, pool, _i(3), _i(3), 4)
    with pytest.raises(ValueError):
        paged.paged_append(x, pool, pool, _i(2), _i(3), 4)
    with pytest.raises(ValueError):
        paged.paged_append(x[:, :-1], pool, pool, _i(3), _i(3), 4)
    with pytest.raises(ValueError):
        paged.paged_append(x, pool, pool.transpose(1, 2).contiguous().transpose(1, 2), _i(3), _i(3), 4)
    with pytest.raises(ValueError):
        paged.paged_append(x, pool, pool, _i(3), _i(3), 4, q_norm=torch.ones(32), k_norm=torch.ones(64))
    with pytest.raises(ValueError):
        paged.paged_append(x, pool, pool, _i(3), _i(3), 4, q_dtype=torch.float16)
    with pytest.raises(ValueError):
        paged.paged_attention(q, pool, pool, _i(2, 3), _i(3), _i(2), 2)
    with pytest.raises(ValueError):
        paged.paged_attention(q, pool, pool, _i(2, 3), _i(2), _i(2), 2)
    with pytest.raises(ValueError):
        paged.paged_attention(q.half(), pool, pool, _i(2, 3), _i(3), _i(2), 2)
    with pytest.raises(ValueError):
        paged.paged_attention(q.transpose(0, 1), pool, pool, _i(2, 3), _i(3), _i(2), 2)
    with pytest.raises(ValueError):
        paged.paged_attention(q, pool.double(), pool.double(), _i(2, 3), _i(3), _i(2), 2)
