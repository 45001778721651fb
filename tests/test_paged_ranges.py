"""Python's integers have no width: sizes that the C calls' 32-bit arguments cannot hold are refused, not cut."""
import pytest

from anetransformers_b200 import SpecDecError, paged
from tests.conftest import gpu_available

BIG = (1 << 32) + 8  # 8 in 32 bits


@pytest.mark.parametrize("name", ["max_q", "max_kv", "prefix_len", "window"])
@pytest.mark.parametrize("value", [BIG, 1 << 31, -1])
def test_attention_sizes(name, value):
    import torch
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    kp, q = torch.zeros(8, 16, 2, 64, dtype=torch.float16), torch.zeros(2, 4, 64, dtype=torch.float16)
    kw = dict(max_q=1, max_kv=16, prefix_len=0, window=0)
    kw[name] = value
    with pytest.raises(SpecDecError, match=name):
        paged.attention_dev(q, kp, kp, i32(2, 4), i32(2), i32(2), i32(2), prefix_table=i32(4), **kw)


@pytest.mark.parametrize("args", [(BIG, 8, 16, 64), (2, BIG, 16, 64), (2, 8, BIG, 64)])
def test_pool_sizes(args):
    with pytest.raises(SpecDecError, match="PagePool"):
        paged.PagePool(*args, device="meta")


@pytest.mark.gpu
@pytest.mark.skipif(not gpu_available(), reason="needs a CUDA GPU")
@pytest.mark.parametrize("kw", [dict(n_tokens=-1), dict(n_tokens=BIG), dict(q_stride=BIG), dict(q_stride=-1), dict(pos0=BIG), dict(pos0=-1)])
def test_plan_sizes(kw):
    import torch
    pool = paged.PagePool(2, 8, 16, 64)
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    a = dict(n_tokens=2, q_stride=0, pos0=0)
    a.update(kw)
    with pytest.raises(SpecDecError, match=next(iter(kw))):
        pool.plan(one, one, **a, out=pool.plan(one, one, 2))
