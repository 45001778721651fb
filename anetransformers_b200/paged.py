"""Paged K/V cache on torch device tensors: pages shared by many requests, and attention over them (sd_pages_*,
sd_kv_append_dev and sd_attention_dev of the C ABI; the rules are in include/specdec_b200.h).

A serving step of a batch::

    pool = PagePool(n_req, n_pages, page_size, max_len)
    step = pool.plan(kv_len, q_len, n_tokens)                    # block tables, slots of the new tokens
    append_dev(k, v, step.slots, k_pages, v_pages)               # their K and V into the pages
    out = attention_dev(q, k_pages, v_pages, pool.table, kv_len, step.q_start, q_len, max_q=..., max_kv=...)

The calls run on the current stream of the tensors' device, and can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional

from . import _lib

_DTYPES = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2}
_ERR_INVALID = -1


def _refuse(msg: str):
    raise _lib.SpecDecError(_ERR_INVALID, msg)


def _i32(name, t, numel=None, contiguous=True):
    if str(t.dtype) != "torch.int32":
        _refuse(f"{name} must be int32, not {t.dtype}")
    if contiguous and not t.is_contiguous():
        _refuse(f"{name} must be contiguous")
    if numel is not None and t.numel() != numel:
        _refuse(f"{name} has {t.numel()} entries, not {numel}")
    return t


class _On:
    """The tensors' device as the current one, and its current stream."""

    def __init__(self, *tensors):
        import torch
        dev = tensors[0].device
        if dev.type != "cuda":
            _refuse("the tensors must be in device memory")
        for t in tensors[1:]:
            if t is not None and t.device != dev:
                _refuse(f"tensors on {t.device} and {dev}")
        self.dev = dev.index
        self.prev = torch.cuda.current_device()
        self.torch = torch

    def __enter__(self):
        if self.prev != self.dev:
            self.torch.cuda.set_device(self.dev)
        return self.torch.cuda.current_stream(self.dev).cuda_stream

    def __exit__(self, *a):
        if self.prev != self.dev:
            self.torch.cuda.set_device(self.prev)


class Plan(NamedTuple):
    """One step's slot map: q_start [n_req], slots and positions [n_tokens], missing [1] pages."""
    q_start: "object"
    slots: "object"
    positions: "object"
    missing: "object"


class PagePool:
    """Which request holds which page: table [n_req, pages of max_len] (-1 behind a request's pages), held [n_req],
    and the stack of free pages (free [n_pages], n_free [1]).  A shared prefix is a request of its own: its row of
    the table is the prefix_table of attention_dev."""

    def __init__(self, n_req: int, n_pages: int, page_size: int, max_len: int, device="cuda"):
        import torch
        if n_req < 1 or n_pages < 1 or max_len < 1 or page_size < 1:
            _refuse(f"PagePool({n_req}, {n_pages}, {page_size}, {max_len})")
        self.page_size = page_size
        self.table = torch.empty(n_req, -(-max_len // page_size), dtype=torch.int32, device=device)
        self.held = torch.empty(n_req, dtype=torch.int32, device=device)
        self.free = torch.empty(n_pages, dtype=torch.int32, device=device)
        self.n_free = torch.empty(1, dtype=torch.int32, device=device)
        self._c = _lib.Pages(self.table.data_ptr(), self.held.data_ptr(), self.free.data_ptr(), self.n_free.data_ptr(),
                             n_req, self.table.shape[1], n_pages, page_size)
        self.reset()

    def reset(self):
        """Every page free, no request holds any."""
        with _On(self.table) as st:
            _lib.check(_lib.lib().sd_pages_reset_dev(C.byref(self._c), st), "pages reset")

    def plan(self, kv_len, q_len, n_tokens: int, q_stride: int = 0, pos0: int = 0, out: Optional[Plan] = None) -> Plan:
        """Pages and slots of one step (sd_pages_plan_dev): kv_len [n_req] positions after it, q_len [n_req] new ones."""
        import torch
        n = self._c.n_req
        _i32("kv_len", kv_len, n), _i32("q_len", q_len, n)
        if out is None:
            buf = torch.empty(n + 2 * n_tokens + 1, dtype=torch.int32, device=self.table.device)
            out = Plan(*buf.split((n, n_tokens, n_tokens, 1)))
        else:
            for name, t, m in zip(out._fields, out, (n, n_tokens, n_tokens, 1)):
                _i32(name, t, m)
        with _On(self.table, kv_len, q_len, *out) as st:
            _lib.check(_lib.lib().sd_pages_plan_dev(C.byref(self._c), kv_len.data_ptr(), q_len.data_ptr(), q_stride, pos0,
                                                    n_tokens, out.q_start.data_ptr(), out.slots.data_ptr(),
                                                    out.positions.data_ptr(), out.missing.data_ptr(), st), "pages plan")
        return out


def _kv_pool(k_pages, v_pages) -> _lib.KvPool:
    """k_pages, v_pages: [n_pages, page_size, n_kv_heads, head_dim] views of the same strides, last dimension dense."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        _refuse(f"pages {tuple(k_pages.shape)} {k_pages.dtype} and {tuple(v_pages.shape)} {v_pages.dtype}")
    st = k_pages.stride()
    if st != v_pages.stride() or st[3] != 1:
        _refuse(f"page strides {st} and {v_pages.stride()}")
    dt = _DTYPES.get(str(k_pages.dtype), -1)
    n, ps, h, d = k_pages.shape
    return _lib.KvPool(k_pages.data_ptr(), v_pages.data_ptr(), st[0], st[1], st[2], n, ps, h, d, dt)


def append_dev(k, v, slots, k_pages, v_pages):
    """k, v [n, n_kv_heads, head_dim] (tokens at any stride, heads dense) into the pages at slots [n] int32."""
    pool = _kv_pool(k_pages, v_pages)
    n = slots.numel()
    for t in (k, v):
        if t.shape != (n, pool.n_kv_heads, pool.head_dim) or t.dtype != k.dtype:
            _refuse(f"rows {tuple(t.shape)} {t.dtype} for {n} slots of [{pool.n_kv_heads}, {pool.head_dim}]")
        if t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != pool.head_dim):
            _refuse("a token's heads must be dense")
    _i32("slots", slots)
    src = _DTYPES.get(str(k.dtype), -1)
    with _On(k_pages, v_pages, k, v, slots) as st:
        _lib.check(_lib.lib().sd_kv_append_dev(C.byref(pool), k.data_ptr(), v.data_ptr(), src, k.stride(0), v.stride(0),
                                               slots.data_ptr(), n, st), "kv append")


def attention_dev(q, k_pages, v_pages, table, kv_len, q_start, q_len, *, max_q: int, max_kv: int, prefix_table=None,
                  prefix_len: int = 0, scale: Optional[float] = None, softcap: float = 0.0, window: int = 0, alibi=None,
                  out=None):
    """q [n_tokens, n_heads, head_dim] (any token and head stride) over the pages -> out, like q (sd_attention_dev).
    table [n_req, m] int32; kv_len, q_start, q_len [n_req] int32; max_q, max_kv: host bounds on q_len and kv_len;
    prefix_table: pages of the prefix_len positions that every request shares; alibi [n_heads] fp32 slopes.
    Tokens of no request are left as out has them."""
    import torch
    pool = _kv_pool(k_pages, v_pages)
    if q.dim() != 3 or q.shape[2] != pool.head_dim or q.dtype != k_pages.dtype or q.stride(2) != 1:
        _refuse(f"q {tuple(q.shape)} {q.dtype} over pages of [{pool.n_kv_heads}, {pool.head_dim}] {k_pages.dtype}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
        _refuse(f"out {tuple(out.shape)} {out.dtype} for q {tuple(q.shape)} {q.dtype}")
    if table.dim() != 2 or table.stride(1) != 1:
        _refuse("table must be [n_req, pages] with dense rows")
    n_req = table.shape[0]
    _i32("table", table, contiguous=False)
    for name, t in (("kv_len", kv_len), ("q_start", q_start), ("q_len", q_len)):
        _i32(name, t, n_req)
    # a one-row table's row stride is free to be anything
    if table.shape[1] * pool.page_size < max_kv:
        _refuse(f"max_kv {max_kv} beyond the table's {table.shape[1]} pages of {pool.page_size}")
    ld = table.stride(0) if n_req > 1 else table.shape[1]
    if prefix_len > 0:
        if prefix_table is None or _i32("prefix_table", prefix_table).numel() * pool.page_size < prefix_len:
            _refuse(f"prefix_table does not hold {prefix_len} positions")
    if alibi is not None and (str(alibi.dtype) != "torch.float32" or alibi.numel() != q.shape[1] or not alibi.is_contiguous()):
        _refuse("alibi must be float32 [n_heads]")
    a = _lib.AttnArgs(pool, q.data_ptr(), out.data_ptr(), q.stride(0), q.stride(1), out.stride(0), out.stride(1),
                      table.data_ptr(), kv_len.data_ptr(), q_start.data_ptr(), q_len.data_ptr(),
                      prefix_table.data_ptr() if prefix_len > 0 else None, alibi.data_ptr() if alibi is not None else None,
                      q.shape[0], q.shape[1], n_req, ld, max_q, max_kv, prefix_len, window,
                      scale if scale is not None else 1.0 / math.sqrt(pool.head_dim), softcap, None, 0)
    L = _lib.lib()
    with _On(q, out, k_pages, v_pages, table, kv_len, q_start, q_len, prefix_table if prefix_len > 0 else None, alibi) as st:
        n = L.sd_attention_workspace(C.byref(a))
        if n:
            ws = torch.empty(n, dtype=torch.uint8, device=q.device)  # of this stream: freed in its order
            a.workspace, a.workspace_bytes = ws.data_ptr(), n
        _lib.check(L.sd_attention_dev(C.byref(a), st), "attention")
    return out
