"""The page plan's checks of what only the device knows: entries out of range are left out and recorded (code 3)."""
import ctypes as C
import threading

import pytest

from tests.conftest import gpu_available
from tests.test_gpu_paged import clean_error_word, error_word, i32, pg  # noqa: F401 (fixtures)

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a CUDA GPU")]

GUARD = 77


class Guarded:
    """A pool of 8 pages of 16 positions whose arrays lie between words that nothing may write."""

    def __init__(self, n_req=2, ld=4, n_pages=8):
        import torch
        from anetransformers_b200 import _lib
        self.sizes = dict(table=n_req * ld, held=n_req, free_pages=n_pages, n_free=1)
        self.mem = {k: torch.full((n + 64,), GUARD, dtype=torch.int32, device="cuda") for k, n in self.sizes.items()}
        self.c = _lib.Pages(*(m[32:].data_ptr() for m in self.mem.values()), n_req, ld, n_pages, 16)
        self.lib = _lib.lib()
        assert self.lib.sd_pages_reset_dev(C.byref(self.c), self.stream()) == 0

    def stream(self):
        import torch
        return torch.cuda.current_stream().cuda_stream

    def __getitem__(self, k):
        return self.mem[k][32:32 + self.sizes[k]]

    def plan(self, kv, q, n_tokens=0):
        a = [i32(kv), i32(q), i32([0] * len(kv)), i32([0] * max(n_tokens, 1)), i32([0])]
        assert self.lib.sd_pages_plan_dev(C.byref(self.c), a[0].data_ptr(), a[1].data_ptr(), 0, 0, n_tokens, a[2].data_ptr(),
                                          a[3].data_ptr(), None, a[4].data_ptr(), self.stream()) == 0
        for k, m in self.mem.items():
            n = self.sizes[k]
            assert bool((m[:32] == GUARD).all()) and bool((m[32 + n:] == GUARD).all()), k
        return a[4].item()


@pytest.mark.parametrize("n_free", [-3, -(1 << 31), -1])
def test_negative_count_of_free_pages(pg, n_free):
    """Taken as an empty stack: pages given back land at its start, and can be taken in the same step."""
    p = Guarded()
    p.plan([60, 1], [0, 0])
    assert error_word() == 0 and p["table"].tolist() == [0, 1, 2, 3, 4, -1, -1, -1]
    p["n_free"].fill_(n_free)
    p.plan([1, 1], [0, 0])
    assert error_word() == 3
    assert p["n_free"].item() == 3 and p["free_pages"].tolist()[:3] == [1, 2, 3]
    p["n_free"].fill_(n_free)
    assert p.plan([1, 60], [0, 0]) == 3          # nothing to take
    assert error_word() == 3
    assert p["held"].tolist() == [1, 1] and p["n_free"].item() == 0


@pytest.mark.parametrize("n_free", [9, 13, (1 << 31) - 1])
def test_more_free_pages_than_pages(pg, n_free):
    """Taken as a full stack; pages given back to it are dropped."""
    p = Guarded()
    p["n_free"].fill_(n_free)
    p.plan([20, 0], [0, 0])
    assert error_word() == 3
    assert p["table"].tolist()[:2] == [0, 1] and p["n_free"].item() == 6
    p["n_free"].fill_(n_free)
    p.plan([1, 0], [0, 0])
    assert error_word() == 3
    assert p["held"].tolist() == [1, 0] and p["n_free"].item() == 8
    p["n_free"].fill_(7)
    p["held"].copy_(i32([3, 0]))                 # two more pages given back than the stack has room for one of
    p.plan([1, 0], [0, 0])
    assert error_word() == 3 and p["n_free"].item() == 8


@pytest.mark.parametrize("held,kept", [(-1, 0), (5, 4), ((1 << 31) - 1, 4)])
def test_pages_held_out_of_range(pg, held, kept):
    p = Guarded()
    p.plan([64, 0], [0, 0])
    p["held"].copy_(i32([held, 0]))
    p["n_free"].fill_(0)
    p.plan([16 * kept, 0], [0, 0])
    assert error_word() == 3
    p["held"].copy_(i32([4, 0]))
    p.plan([64, 0], [0, 0])
    assert error_word() == 0


def test_page_ids_out_of_the_pool(pg):
    """A free stack that names pages that do not exist: no slot is made of them."""
    pool = pg.PagePool(2, 8, 16, 64)
    pool.free[6:] = i32([8, 1 << 28])  # the next two pages taken: 2^28 (whose slots would wrap to 0 and on), then 8
    got = pool.plan(i32([3, 18]), i32([3, 18]), 21)  # request 1 gets page 8, which is none, then free[5] = 2
    assert error_word() == 3
    assert got.slots.tolist() == [-1] * 19 + [2 * 16, 2 * 16 + 1]
    assert got.positions.tolist() == list(range(3)) + list(range(18))


def test_more_new_tokens_than_32_bits_count(pg):
    """Lengths that add up past 2^31: the tokens that have room are those of the first requests, the others are dropped."""
    n, room = 4096, 1 << 20
    pool = pg.PagePool(n, 64, 16, 64)
    got = pool.plan(i32([5] + [0] * (n - 1)), i32([5] + [room] * (n - 1)), room)
    assert error_word() == 3
    assert got.positions[:5].tolist() == list(range(5)) and got.slots[:5].tolist() == list(range(5))
    assert bool((got.slots[5:] == -1).all())
    assert got.q_start[:3].tolist() == [0, 5, 5 + room]


def test_large_batches_from_two_threads(pg):
    """Two host threads that plan large batches of different sizes, each on a pool and a stream of its own."""
    import torch
    from anetransformers_b200 import _lib
    plan, failed = _lib.lib().sd_pages_plan_dev, []

    def loop(n):
        with torch.cuda.stream(torch.cuda.Stream()):
            pool = pg.PagePool(n, n, 16, 16)
            kv, q, q_start = i32([1] * n), i32([0] * n), i32([0] * n)
            c = _lib.Pages(pool.table.data_ptr(), pool.held.data_ptr(), pool.free.data_ptr(), pool.n_free.data_ptr(), n, 1, n, 16)
            args = (C.byref(c), kv.data_ptr(), q.data_ptr(), 0, 0, 0, q_start.data_ptr(), None, None, None,
                    torch.cuda.current_stream().cuda_stream)
            failed.extend(rc for rc in (plan(*args) for _ in range(20000)) if rc)
            torch.cuda.current_stream().synchronize()
            failed.extend(x for x in pool.held.tolist() if x != 1)
    threads = [threading.Thread(target=loop, args=(n,)) for n in (4096, 3100)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
