"""A context of nearly 2^31 positions, the most that a block table can name: its pages are all the same one but the last."""
import pytest

from tests.conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a CUDA GPU")]


@pytest.mark.parametrize("behind", [0, 100, 70000, 1 << 20])
def test_last_page_of_the_longest_context(behind):
    """The only keys with a score (40) lie in one page `behind` positions before the end: the rows' output is their V, 1.
    The other keys weigh 2^31 e^-40 = 9.2e-9 of one of them, and have V = 0."""
    import torch
    from anetransformers_b200 import paged
    page, hk, hd = 256, 8, 64
    kv = (1 << 31) - 2048
    kp, vp = (torch.zeros(2, page, hk, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    kp[1, ..., 0], vp[1] = 8.0, 1.0
    table = torch.zeros(1, kv // page, dtype=torch.int32, device="cuda")
    table[0, (kv - 1 - behind) // page] = 1
    q = torch.zeros(1, hk, hd, dtype=torch.float16, device="cuda")
    q[..., 0] = 5.0
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    out = paged.attention_dev(q, kp, vp, table, i32([kv]), i32([0]), i32([1]), max_q=1, max_kv=kv, scale=1.0)
    assert out.flatten().tolist() == [1.0] * (hk * hd)
