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

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ERR_INVALID = -1


def _refuse(msg: str):
    raise _lib.SpecDecError(_ERR_INVALID, msg)


def _sizes(**kw):
    """Sizes as the C calls take them: ctypes would cut a wider integer to its low 32 bits."""
    for name, v in kw.items():
        if not 0 <= v <= 0x7FFFFFFF:
            _refuse(f"{name} {v} outside 0..2^31-1")


def _i32(name, t, numel=None):
    if t.dtype is not torch.int32:
        _refuse(f"{name} must be int32, not {t.dtype}")
    if not t.is_contiguous():
        _refuse(f"{name} must be contiguous")
    if numel is not None and t.numel() != numel:
        _refuse(f"{name} has {t.numel()} entries, not {numel}")
    return t.data_ptr()


def _call(what, fn, tensors, *args):
    """fn(*args, stream) with the tensors' device as the current one, on its current stream."""
    dev = tensors[0].get_device()
    if dev < 0:
        _refuse("the tensors must be in device memory")
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _refuse(f"tensors on {t.device} and {tensors[0].device}")
    stream = torch.cuda.current_stream(dev).cuda_stream
    if torch.cuda.current_device() == dev:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc, what)


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
        if not all(1 <= x <= 0x7FFFFFFF for x in (n_req, n_pages, page_size, max_len)):
            _refuse(f"PagePool({n_req}, {n_pages}, {page_size}, {max_len})")
        self.page_size = page_size
        self.table = torch.empty(n_req, -(-max_len // page_size), dtype=torch.int32, device=device)
        self.held = torch.empty(n_req, dtype=torch.int32, device=device)
        self.free = torch.empty(n_pages, dtype=torch.int32, device=device)
        self.n_free = torch.empty(1, dtype=torch.int32, device=device)
        self._c = _lib.Pages(self.table.data_ptr(), self.held.data_ptr(), self.free.data_ptr(), self.n_free.data_ptr(),
                             n_req, self.table.shape[1], n_pages, page_size)
        self._ref = C.byref(self._c)
        self.reset()

    def reset(self):
        """Every page free, no request holds any."""
        _call("pages reset", _lib.lib().sd_pages_reset_dev, (self.table,), self._ref)

    def plan(self, kv_len, q_len, n_tokens: int, q_stride: int = 0, pos0: int = 0, out: Optional[Plan] = None) -> Plan:
        """Pages and slots of one step (sd_pages_plan_dev): kv_len [n_req] positions after it, q_len [n_req] new ones."""
        n, dev = self._c.n_req, self.table.device
        _sizes(n_tokens=n_tokens, q_stride=q_stride, pos0=pos0)
        if out is None:
            buf = torch.empty(n + 2 * n_tokens + 1, dtype=torch.int32, device=dev)
            out = Plan(*buf.split_with_sizes((n, n_tokens, n_tokens, 1)))
        _call("pages plan", _lib.lib().sd_pages_plan_dev, (self.table, kv_len, q_len, *out), self._ref, _i32("kv_len", kv_len, n),
              _i32("q_len", q_len, n), q_stride, pos0, n_tokens, _i32("q_start", out.q_start, n), _i32("slots", out.slots, n_tokens),
              _i32("positions", out.positions, n_tokens), _i32("missing", out.missing, 1))
        return out


def _kv_pool(k_pages, v_pages) -> _lib.KvPool:
    """k_pages, v_pages: [n_pages, page_size, n_kv_heads, head_dim] views of the same strides, last dimension dense."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        _refuse(f"pages {tuple(k_pages.shape)} {k_pages.dtype} and {tuple(v_pages.shape)} {v_pages.dtype}")
    st = k_pages.stride()
    if st != v_pages.stride() or st[3] != 1:
        _refuse(f"page strides {st} and {v_pages.stride()}")
    dt = _DTYPES.get(k_pages.dtype, -1)
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
    _call("kv append", _lib.lib().sd_kv_append_dev, (k_pages, v_pages, k, v, slots), C.byref(pool), k.data_ptr(), v.data_ptr(),
          _DTYPES.get(k.dtype, -1), k.stride(0), v.stride(0), _i32("slots", slots), n)


def attention_dev(q, k_pages, v_pages, table, kv_len, q_start, q_len, *, max_q: int, max_kv: int, prefix_table=None,
                  prefix_len: int = 0, scale: Optional[float] = None, softcap: float = 0.0, window: int = 0, alibi=None,
                  out=None):
    """q [n_tokens, n_heads, head_dim] (any token and head stride) over the pages -> out, like q (sd_attention_dev).
    table [n_req, m] int32; kv_len, q_start, q_len [n_req] int32; max_q, max_kv: host bounds on q_len and kv_len;
    prefix_table: pages of the prefix_len positions that every request shares; alibi [n_heads] fp32 slopes.
    Tokens of no request are left as out has them."""
    pool = _kv_pool(k_pages, v_pages)
    _sizes(max_q=max_q, max_kv=max_kv, prefix_len=prefix_len, window=window)
    if q.dim() != 3 or q.shape[2] != pool.head_dim or q.dtype is not k_pages.dtype or q.stride(2) != 1:
        _refuse(f"q {tuple(q.shape)} {q.dtype} over pages of [{pool.n_kv_heads}, {pool.head_dim}] {k_pages.dtype}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype is not q.dtype or out.stride(2) != 1:
        _refuse(f"out {tuple(out.shape)} {out.dtype} for q {tuple(q.shape)} {q.dtype}")
    if table.dim() != 2 or table.stride(1) != 1 or table.dtype is not torch.int32:
        _refuse("table must be int32 [n_req, pages] with dense rows")
    n_req = table.shape[0]
    if table.shape[1] * pool.page_size < max_kv:
        _refuse(f"max_kv {max_kv} beyond the table's {table.shape[1]} pages of {pool.page_size}")
    # a one-row table's row stride is free to be anything
    ld = table.stride(0) if n_req > 1 else table.shape[1]
    prefix = None
    if prefix_len > 0:
        prefix = _i32("prefix_table", prefix_table) if prefix_table is not None else 0
        if not prefix or prefix_table.numel() * pool.page_size < prefix_len:
            _refuse(f"prefix_table does not hold {prefix_len} positions")
    if alibi is not None and (alibi.dtype is not torch.float32 or alibi.numel() != q.shape[1] or not alibi.is_contiguous()):
        _refuse("alibi must be float32 [n_heads]")
    qs, os = q.stride(), out.stride()
    a = _lib.AttnArgs(pool, q.data_ptr(), out.data_ptr(), qs[0], qs[1], os[0], os[1], table.data_ptr(), _i32("kv_len", kv_len, n_req),
                      _i32("q_start", q_start, n_req), _i32("q_len", q_len, n_req), prefix,
                      alibi.data_ptr() if alibi is not None else None, q.shape[0], q.shape[1], n_req, ld, max_q, max_kv, prefix_len,
                      window, scale if scale is not None else 1.0 / math.sqrt(pool.head_dim), softcap, None, 0)
    L, ref = _lib.lib(), C.byref(a)
    n = L.sd_attention_workspace(ref)
    if n:
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)  # of this stream: freed in its order
        a.workspace, a.workspace_bytes = ws.data_ptr(), n
    _call("attention", L.sd_attention_dev, (q, out, k_pages, v_pages, table, kv_len, q_start, q_len,
                                            prefix_table if prefix_len > 0 else None, alibi), ref)
    return out
