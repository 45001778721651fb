"""Steps without a token (every request idle): nothing to do, and no pointer to rows that are not there is asked for."""
import ctypes as C

import pytest

from anetransformers_b200 import _lib
from tests.conftest import gpu_available
from tests.test_paged import P, attn, pool, refused


def test_no_rows_no_pointers():
    L = _lib.lib()
    assert L.sd_kv_append_dev(C.byref(pool()), None, None, 0, 0, 0, None, 0, None) == 0
    assert L.sd_attention_dev(C.byref(attn(n_tokens=0, q=None, out=None)), None) == 0
    assert L.sd_attention_workspace(C.byref(attn(n_tokens=0, q=None, out=None))) == 0
    refused(L.sd_kv_append_dev(C.byref(pool(k=None)), None, None, 0, 0, 0, None, 0, None))
    refused(L.sd_attention_dev(C.byref(attn(n_tokens=0, q=None, out=None, kv_len=None)), None))
    refused(L.sd_kv_append_dev(C.byref(pool()), None, P, 0, 1024, 1024, P, 1, None))
    refused(L.sd_attention_dev(C.byref(attn(n_tokens=1, q=None)), None))


@pytest.mark.gpu
@pytest.mark.skipif(not gpu_available(), reason="needs a CUDA GPU")
def test_a_step_without_tokens():
    import torch
    from anetransformers_b200 import paged
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    pages = paged.PagePool(2, 8, 16, 64)
    kv = i32([20, 3])
    pages.plan(kv, kv, 23)
    step = pages.plan(kv, i32([0, 0]), 0)
    kp = torch.ones(8, 16, 2, 64, dtype=torch.float16, device="cuda")
    vp = kp.clone()
    rows, q = torch.zeros(5, 2, 64, device="cuda"), torch.zeros(5, 4, 64, dtype=torch.float16, device="cuda")
    paged.append_dev(rows[:0], rows[5:], step.slots, kp, vp)
    assert bool((kp == 1).all()) and bool((vp == 1).all())
    out = paged.attention_dev(q[:0], kp, vp, pages.table, kv, step.q_start, i32([0, 0]), max_q=0, max_kv=64)
    assert out.shape == (0, 4, 64)
    out = paged.attention_dev(q[:0], kp, vp, pages.table, kv, step.q_start, i32([0, 0]), max_q=4, max_kv=64, out=q[:0])
    assert out.shape == (0, 4, 64)
    assert pages.held.tolist() == [2, 1] and _lib.lib().sd_device_error(0) == 0
