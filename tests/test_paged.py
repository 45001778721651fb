"""Refusals of the paged K/V cache operators (host-side argument checks: no GPU is touched) and the tests' own
restatement of the page plan."""
import ctypes as C

import pytest

from anetransformers_b200 import _lib
from tests import paged_oracle as PO

P = 4096  # a pointer that is never read: every call below is refused before it looks at one


def pages(**kw):
    a = dict(table=P, held=P, free_pages=P, n_free=P, n_req=4, table_ld=8, n_pages=64, page_size=16)
    a.update(kw)
    return _lib.Pages(**a)


def pool(**kw):
    a = dict(k=P, v=P, page_stride=16 * 8 * 128, pos_stride=8 * 128, head_stride=128, n_pages=64, page_size=16, n_kv_heads=8,
             head_dim=128, dtype=1)
    a.update(kw)
    return _lib.KvPool(**a)


def attn(pool_kw=None, **kw):
    a = dict(pool=pool(**(pool_kw or {})), q=P, out=P, q_ld=4096, q_head=128, out_ld=4096, out_head=128, table=P, kv_len=P,
             q_start=P, q_len=P, prefix_table=None, alibi=None, n_tokens=4, n_heads=32, n_req=4, table_ld=8, max_q=1, max_kv=128,
             prefix_len=0, window=0, scale=0.1, softcap=0.0, workspace=None, workspace_bytes=0)
    a.update(kw)
    return _lib.AttnArgs(**a)


def refused(rc, word=None):
    assert rc == -1, rc  # SD_ERR_INVALID
    msg = _lib.last_error()
    assert msg and (word is None or word in msg), msg


@pytest.mark.parametrize("kw", [dict(table=None), dict(held=None), dict(free_pages=None), dict(n_free=None), dict(n_req=0),
                                dict(n_req=4097), dict(table_ld=0), dict(n_pages=0), dict(page_size=8), dict(page_size=48),
                                dict(page_size=512), dict(n_pages=1 << 28), dict(table_ld=1 << 28), dict(n_req=4096, table_ld=1 << 20)])
def test_pages_refusals(kw):
    L = _lib.lib()
    p = pages(**kw)
    refused(L.sd_pages_plan_dev(C.byref(p), P, P, 0, 0, 4, P, P, None, None, None))
    refused(L.sd_pages_reset_dev(C.byref(p), None))


@pytest.mark.parametrize("args", [(None, P, 0, 0, 4, P, P), (P, None, 0, 0, 4, P, P), (P, P, 0, 0, 4, None, P),
                                  (P, P, 0, 0, 4, P, None), (P, P, -1, 0, 4, P, P), (P, P, 0, -1, 4, P, P), (P, P, 0, 0, -1, P, P),
                                  (P, P, 1 << 30, 0, 4, P, P), (P, P, 0, (1 << 31) - 64, 4, P, P)])
def test_plan_refusals(args):
    p = pages()
    refused(_lib.lib().sd_pages_plan_dev(C.byref(p), *args, None, None, None))


@pytest.mark.parametrize("kw", [dict(k=None), dict(v=None), dict(page_size=17), dict(n_pages=0), dict(n_kv_heads=0), dict(head_dim=12),
                                dict(head_dim=264), dict(dtype=0), dict(dtype=3), dict(head_stride=64), dict(pos_stride=0)])
def test_pool_refusals(kw):
    L = _lib.lib()
    p = pool(**kw)
    refused(L.sd_kv_append_dev(C.byref(p), P, P, 0, 1024, 1024, P, 4, None))
    refused(L.sd_attention_dev(C.byref(attn(kw)), None))


def test_append_refusals():
    L, p = _lib.lib(), pool()
    refused(L.sd_kv_append_dev(C.byref(p), None, P, 0, 1024, 1024, P, 4, None))
    refused(L.sd_kv_append_dev(C.byref(p), P, P, 2, 1024, 1024, P, 4, None), "type")   # bf16 rows, fp16 pool
    refused(L.sd_kv_append_dev(C.byref(p), P, P, 0, 1024, 1024, None, 4, None))
    refused(L.sd_kv_append_dev(C.byref(p), P, P, 0, 1024, 1024, P, -1, None))


@pytest.mark.parametrize("kw", [dict(q=None), dict(out=None), dict(table=None), dict(kv_len=None), dict(q_start=None), dict(q_len=None),
                                dict(n_req=0), dict(n_req=4097), dict(n_heads=0), dict(n_heads=30), dict(n_heads=8 * 129), dict(max_kv=129),
                                dict(max_q=-1), dict(max_kv=-1), dict(n_tokens=-1), dict(prefix_len=-1), dict(prefix_len=16),
                                dict(window=-1), dict(table_ld=0), dict(softcap=-1.0), dict(softcap=float("nan")),
                                dict(scale=float("nan")), dict(scale=float("inf")), dict(softcap=1e-9), dict(softcap=float("inf")), dict(q_head=64), dict(out_head=64),
                                dict(prefix_len=(1 << 31) - 600, prefix_table=P)])
def test_attention_refusals(kw):
    refused(_lib.lib().sd_attention_dev(C.byref(attn(**kw)), None))


def test_nothing_to_do():
    """No tokens: no launch, no error, also without a GPU."""
    assert _lib.lib().sd_attention_dev(C.byref(attn(n_tokens=0)), None) == 0
    assert _lib.lib().sd_kv_append_dev(C.byref(pool()), P, P, 0, 1024, 1024, P, 0, None) == 0


def test_plan_oracle_rules():
    """The restatement the GPU tests compare with, on a step small enough to follow by hand (pages of 16)."""
    st = dict(table=[[], [], []], free=[4, 3, 2, 1, 0], ld=4)
    assert PO.plan(st, [17, 1, 16], [17, 1, 16], 16, 40)[3] == 0
    assert st["table"] == [[0, 1], [2], [3]] and st["free"] == [4]
    # request 0 shrinks to one page, request 1 grows by two, request 2 ends
    q_start, slots, pos, missing = PO.plan(st, [16, 40, 0], [1, 2, 0], 16, 4, pos0=100)
    assert st["table"] == [[0], [2, 3, 1], []] and st["free"] == [4] and missing == 0
    assert q_start == [0, 1, 3] and slots == [15, 1 * 16 + 6, 1 * 16 + 7, -1] and pos == [115, 138, 139, -1]
    # two pages wanted, one free
    q_start, slots, pos, missing = PO.plan(st, [16, 40, 17], [0, 0, 2], 16, 2)
    assert missing == 1 and st["table"][2] == [4] and slots == [4 * 16 + 15, -1] and pos == [15, 16]


def test_shared_batch_refusals():
    L, out = _lib.lib(), C.c_void_p()
    for args in [(None, P, 4, 2, 64, 5), (P, None, 4, 2, 64, 5), (P, P, 0, 2, 64, 5), (P, P, 4, 0, 64, 5), (P, P, 4, 2, 15, 5),
                 (P, P, 4, 2, 64, 0), (P, P, 4, 2, 64, 9), (P, P, 1 << 30, 2, 64, 5)]:
        refused(L.sd_batch_create_shared(*args, C.byref(out)))
    refused(L.sd_batch_create_shared(P, P, 4, 2, 64, 5, None))


@pytest.mark.parametrize("out_ld", [0, 64, 127])
def test_out_rows_that_overlap(out_ld):
    refused(_lib.lib().sd_attention_dev(C.byref(attn(out_ld=out_ld, n_tokens=2)), None), "overlap")
