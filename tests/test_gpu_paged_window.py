"""Windows over the paged cache: K and V that no row sees may hold anything, and pages of which no row sees a position may
be gone, in the prefix as well, however far behind it the requests are."""
import pytest

from tests.conftest import gpu_available
from tests.test_gpu_paged import check_attention, clean_error_word, error_word, make_case, pg  # noqa: F401 (fixtures)

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a CUDA GPU")]

# kv_len, q_len, prefix, window: few rows per kv head; up to two row tiles (prefix items over several requests); one
# request that takes the prefix tiles in front of its own; rows without a position in each
SHAPES = [([400, 420], [1, 2], 600, 500), ([900, 405, 700], [1, 3, 2], 2000, 500), ([400, 0, 430], [40, 0, 30], 600, 500),
          ([70, 90], [100, 1], 300, 120), ([70], [100], 300, 120), ([30, 200], [45, 1], 300, 120), ([2, 500], [4, 1], 700, 90),
          ([300, 301], [250, 200], 400, 350)]


def first_seen(c, window):
    """First prefix position that some row sees."""
    own = [max(0, k - q) for k, q in zip(c["kv_len"].tolist(), c["q_len"].tolist()) if k > 0 and q > 0]
    return min(c["prefix_len"], max(0, c["prefix_len"] + min(own) + 1 - window))


@pytest.mark.parametrize("kv,q,prefix,window", SHAPES)
@pytest.mark.parametrize("hd,page,gap", [(128, 16, 0), (64, 64, 0), (64, 32, 5), (128, 256, 3)])
def test_unseen_prefix_may_hold_anything(pg, kv, q, prefix, window, hd, page, gap):
    import torch
    c = make_case(kv, q, 8, 2, hd, page, "float16", prefix=prefix, seed=prefix + len(kv), gap=gap)
    p = torch.arange(first_seen(c, window))
    assert len(p) > 0
    at = (c["prefix_table"][p // page].long(), p % page)
    c["k_pages"][at] = float("nan")
    c["v_pages"][at] = float("inf")
    check_attention(pg, c, dict(window=window))


@pytest.mark.parametrize("kv,q,prefix,window", SHAPES)
@pytest.mark.parametrize("page", [16, 64])
def test_gone_pages_are_no_error(pg, kv, q, prefix, window, page):
    """Every page behind all rows' windows is -1: the same result, and nothing is recorded."""
    c = make_case(kv, q, 8, 2, 128, page, "bfloat16", prefix=prefix, seed=prefix + len(kv))
    c["prefix_table"][:first_seen(c, window) // page] = -1
    for b, (k, n) in enumerate(zip(kv, q)):
        c["table"][b, :max(0, max(0, k - n) + 1 - window) // page] = -1
    check_attention(pg, c, dict(window=window))
    assert error_word() == 0


@pytest.mark.parametrize("heads,hk", [(2, 2), (8, 1)])
def test_many_requests(pg, heads, hk):
    """More requests than the kernel looks at one by one: several row tiles, each with a least position of its own."""
    import numpy as np
    import torch
    rng = np.random.default_rng(heads)
    n, prefix, window = 600, 500, 300
    kv = rng.integers(130, 180, n).tolist()
    q = [int(x) for x in rng.integers(0, 3, n)]
    c = make_case(kv, q, heads, hk, 64, 16, "float16", prefix=prefix, seed=heads)
    p = torch.arange(first_seen(c, window))
    at = (c["prefix_table"][p // 16].long(), p % 16)
    c["k_pages"][at] = float("nan")
    c["v_pages"][at] = float("inf")
    c["prefix_table"][:len(p) // 16] = -1
    check_attention(pg, c, dict(window=window))
    assert error_word() == 0
