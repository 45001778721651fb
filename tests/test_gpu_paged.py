"""Paged K/V cache on the GPU against plain restatements (tests/paged_oracle.py): page plans and appended rows exactly,
attention within the bound that its oracle derives element by element in 64 bits."""
import math

import numpy as np
import pytest

from tests import paged_oracle as PO
from tests.conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a CUDA GPU")]


@pytest.fixture(scope="module")
def pg():
    from anetransformers_b200 import paged
    return paged


@pytest.fixture(autouse=True)
def clean_error_word():
    from anetransformers_b200 import _lib
    _lib.lib().sd_device_error(0)
    yield
    assert _lib.lib().sd_device_error(0) == 0, "a call recorded an entry out of range"


def error_word():
    from anetransformers_b200 import _lib
    return _lib.lib().sd_device_error(0)


def i32(v):
    import torch
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------------------------------------------
# Page plan
# ---------------------------------------------------------------------------------------------------------------
def check_plan(pool, st, kv, q, page, n_tokens, q_stride=0, pos0=0, got=None):
    got = got or pool.plan(i32(kv), i32(q), n_tokens, q_stride, pos0)
    q_start, slots, pos, missing = PO.plan(st, kv, q, page, n_tokens, q_stride, pos0)
    ld = pool.table.shape[1]
    assert got.q_start.tolist() == q_start
    assert got.slots.tolist() == slots
    assert got.positions.tolist() == pos
    assert got.missing.tolist() == [missing]
    assert pool.table.tolist() == [r + [-1] * (ld - len(r)) for r in st["table"]]
    assert pool.held.tolist() == [len(r) for r in st["table"]]
    assert pool.n_free.tolist() == [len(st["free"])]
    assert pool.free.tolist() == st["free"] + [-1] * (pool.free.numel() - len(st["free"]))


def new_state(n_req, n_pages, ld):
    return dict(table=[[] for _ in range(n_req)], free=list(range(n_pages - 1, -1, -1)), ld=ld)


@pytest.mark.parametrize("n_req,page,max_len,n_pages,q_stride", [(1, 16, 100, 7, 0), (1, 256, 1, 1, 0), (7, 32, 500, 60, 0), (7, 16, 333, 40, 9),
                                                                 (600, 16, 200, 4000, 0), (513, 64, 1000, 5000, 3), (4096, 16, 64, 10000, 0)])
def test_plan_random_steps(pg, n_req, page, max_len, n_pages, q_stride):
    """Requests grow, shrink (rejected drafts), end and are replaced; some steps want more pages than there are."""
    rng = np.random.default_rng(n_req + page)
    pool = pg.PagePool(n_req, n_pages, page, max_len)
    st = new_state(n_req, n_pages, pool.table.shape[1])
    kv = np.zeros(n_req, int)
    for step in range(8):
        grow = rng.integers(0, q_stride + 1 if q_stride else 12, n_req)
        if step == 3 and not q_stride:
            grow[rng.integers(n_req)] = max_len  # one long prompt
        kind = rng.integers(0, 8, n_req)
        kv = np.where(kind == 0, 0, np.where(kind == 1, np.maximum(kv - rng.integers(0, 9, n_req), 0), kv))
        q = np.minimum(np.where(kind == 0, 0, grow), max_len - kv)
        kv = kv + q
        n_tokens = n_req * q_stride if q_stride else int(q.sum()) + int(rng.integers(0, 5))
        check_plan(pool, st, kv.tolist(), q.tolist(), page, n_tokens, q_stride, pos0=17 * step)


def test_plan_ending_and_idle_requests(pg):
    pool = pg.PagePool(3, 8, 16, 64)
    st = new_state(3, 8, 4)
    check_plan(pool, st, [64, 0, 33], [64, 0, 33], 16, 97)
    check_plan(pool, st, [64, 0, 33], [0, 0, 0], 16, 0)       # q_len 0 keeps the pages
    check_plan(pool, st, [0, 40, 33], [0, 40, 0], 16, 48)     # given back and taken in one step, last first
    check_plan(pool, st, [0, 0, 0], [0, 0, 0], 16, 3)
    pool.reset()
    check_plan(pool, new_state(3, 8, 4), [1, 1, 1], [1, 1, 1], 16, 3)


def test_plan_lengths_out_of_range(pg):
    """Cut as documented, recorded in the error word."""
    pool = pg.PagePool(2, 16, 16, 64)
    got = pool.plan(i32([100, 5]), i32([2, 2]), 4)
    assert error_word() == 3
    assert pool.held.tolist() == [4, 1] and got.positions.tolist() == [62, 63, 3, 4]
    got = pool.plan(i32([-5, 3]), i32([0, 4]), 4)       # more new tokens than positions
    assert error_word() == 3
    assert pool.held.tolist() == [0, 1] and got.positions.tolist() == [-1, 0, 1, 2] and got.slots.tolist()[0] == -1
    got = pool.plan(i32([9, 3]), i32([9, 3]), 10)       # 12 tokens, room for 10
    assert error_word() == 3
    assert got.positions.tolist() == list(range(9)) + [0]
    got = pool.plan(i32([9, 3]), i32([4, 3]), 6, q_stride=3)
    assert error_word() == 3
    assert got.q_start.tolist() == [0, 3] and got.positions.tolist() == [6, 7, 8, 0, 1, 2]
    huge = (1 << 31) - 1
    pool.plan(i32([huge, huge]), i32([huge, huge]), 8)
    assert error_word() == 3
    assert pool.held.tolist() == [4, 4]


def test_plan_in_a_graph(pg):
    """One captured plan, replayed with lengths that change in place."""
    import torch
    n, page = 40, 16
    pool = pg.PagePool(n, 600, page, 400)
    st = new_state(n, 600, 25)
    kv, q = i32([0] * n), i32([0] * n)
    out = pool.plan(kv, q, 128)  # empty step; also loads the kernel
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pool.plan(kv, q, 128, out=out)
    rng = np.random.default_rng(4)
    lens = np.zeros(n, int)
    for _ in range(5):
        new = rng.integers(0, 4, n)
        lens = np.where(rng.random(n) < 0.2, 0, lens)
        lens = lens + new
        kv.copy_(i32(lens.tolist()))
        q.copy_(i32(new.tolist()))
        g.replay()
        torch.cuda.synchronize()
        check_plan(pool, st, lens.tolist(), new.tolist(), page, 128, got=out)


def test_python_refusals(pg):
    import torch
    from anetransformers_b200 import SpecDecError
    pool = pg.PagePool(2, 8, 16, 64)
    ok = i32([1, 1])
    kp = torch.zeros(8, 16, 2, 64, dtype=torch.float16, device="cuda")
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda")
    k = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")

    def att(**kw):
        a = dict(q=q, k_pages=kp, v_pages=kp, table=pool.table, kv_len=ok, q_start=ok, q_len=ok, max_q=1, max_kv=16)
        a.update(kw)
        return pg.attention_dev(a.pop("q"), a.pop("k_pages"), a.pop("v_pages"), a.pop("table"), a.pop("kv_len"), a.pop("q_start"),
                                a.pop("q_len"), **a)
    bad = [lambda: pool.plan(ok.long(), ok, 2), lambda: pool.plan(ok, i32([1]), 2), lambda: pool.plan(ok.cpu(), ok, 2),
           lambda: pg.PagePool(2, 8, 24, 64), lambda: pg.PagePool(0, 8, 16, 64),
           lambda: pg.append_dev(k, k[:, :1], ok, kp, kp), lambda: pg.append_dev(k, k, ok.long(), kp, kp),
           lambda: pg.append_dev(k.bfloat16(), k.bfloat16(), ok, kp, kp), lambda: pg.append_dev(k.cpu(), k.cpu(), ok, kp, kp),
           lambda: pg.append_dev(k, k, ok, kp, kp.bfloat16()), lambda: pg.append_dev(k.transpose(0, 1), k, ok, kp, kp),
           lambda: att(q=q.bfloat16()), lambda: att(q=q[:, :3]), lambda: att(max_kv=65), lambda: att(kv_len=ok.long()),
           lambda: att(prefix_len=20, prefix_table=i32([1])), lambda: att(prefix_len=1), lambda: att(alibi=torch.zeros(4, device="cuda").half()),
           lambda: att(softcap=-1.0), lambda: att(k_pages=kp.cpu()), lambda: att(out=q.bfloat16()), lambda: att(table=pool.table.t()),
           lambda: att(k_pages=kp.float(), v_pages=kp.float(), q=q.float())]
    for i, f in enumerate(bad):
        with pytest.raises(SpecDecError):
            f()
            pytest.fail(f"call {i} was not refused")


# ---------------------------------------------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("src,dst,n,hk,hd,page,layout", [
    ("float32", "float16", 1, 8, 128, 16, "nhd"), ("float32", "bfloat16", 37, 8, 128, 64, "nhd"), ("float16", "float16", 320, 2, 64, 16, "hnd"),
    ("bfloat16", "bfloat16", 1000, 8, 128, 256, "pair"), ("bfloat16", "bfloat16", 5, 1, 8, 32, "nhd"), ("float32", "float16", 33, 3, 72, 16, "odd"),
    ("float16", "float16", 33, 3, 72, 16, "odd"), ("bfloat16", "bfloat16", 2, 5, 256, 128, "hnd")])
def test_append(pg, src, dst, n, hk, hd, page, layout):
    """Rounded copies at the slots, every other element as it was; -1 is skipped.  Sources are slices of wider rows."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(n)
    S, D = getattr(torch, src), getattr(torch, dst)
    n_pages = -(-n // page) + 3
    if layout == "hnd":
        kp, vp = (torch.randn(n_pages, hk, page, hd, device="cuda", generator=g).to(D).transpose(1, 2) for _ in range(2))
    elif layout == "pair":
        both = torch.randn(n_pages, 2, page, hk, hd, device="cuda", generator=g).to(D)
        kp, vp = both[:, 0], both[:, 1]
    elif layout == "odd":  # rows one element apart from any alignment
        flat = torch.randn(2, n_pages * page * (hk * hd + 1) + 1, device="cuda", generator=g).to(D)
        kp, vp = (f[1:].view(n_pages, page, hk * hd + 1)[..., :hk * hd].unflatten(2, (hk, hd)) for f in flat)
    else:
        kp, vp = (torch.randn(n_pages, page, hk, hd, device="cuda", generator=g).to(D) for _ in range(2))
    wide = torch.randn(n, 3 * hk * hd + (1 if layout == "odd" else 0), device="cuda", generator=g).to(S)
    k, v = (wide[:, i * hk * hd:(i + 1) * hk * hd].unflatten(1, (hk, hd)) for i in (1, 2))
    slots = torch.randperm(n_pages * page, device="cuda", generator=g)[:n].to(torch.int32)
    slots[n // 2] = -1
    want = []
    for p, r in ((kp, k), (vp, v)):
        w = p.clone()
        ok = slots >= 0
        w[(slots[ok] // page).long(), (slots[ok] % page).long()] = r[ok].to(D)
        want.append(w)
    pg.append_dev(k, v, slots, kp, vp)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


def test_append_bad_slots(pg):
    import torch
    kp, vp = torch.zeros(4, 16, 2, 64, dtype=torch.float16, device="cuda"), torch.zeros(4, 16, 2, 64, dtype=torch.float16, device="cuda")
    k = torch.ones(4, 2, 64, device="cuda")
    pg.append_dev(k, k, i32([-7, 64, 1 << 30, 63]), kp, vp)
    assert error_word() == 3
    assert float(kp.sum()) == 128 and float(vp[3, 15].sum()) == 128


# ---------------------------------------------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------------------------------------------
def make_case(kv, q, heads, hk, hd, page, dtype, prefix=0, seed=0, gap=0, spare=2, sharp=2.0, poison=True):
    """Random pages in random order; positions past every request's end, and the pages of nobody, hold NaN."""
    import torch
    g = torch.Generator().manual_seed(seed)
    D = getattr(torch, dtype)
    nb = [-(-x // page) for x in kv]
    npb = -(-prefix // page)
    n_pages = sum(nb) + npb + spare
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    ld = max(nb + [1]) + 1
    table = torch.full((len(kv), ld), -1, dtype=torch.int32)
    at = npb
    for b, m in enumerate(nb):
        table[b, :m] = order[at:at + m]
        at += m
    kp, vp = (torch.randn(n_pages, page, hk, hd, generator=g).to(D) for _ in range(2))
    if poison:
        used = torch.zeros(n_pages * page, dtype=torch.bool)
        for row, n in [(order[:npb], prefix)] + [(table[b], x) for b, x in enumerate(kv)]:
            p = torch.arange(n)
            used[row[p // page].long() * page + p % page] = True
        for pool, bad in ((kp, float("nan")), (vp, float("inf"))):
            pool.view(n_pages * page, hk, hd)[~used] = bad
    starts, n = [], 0
    for x in q:
        starts.append(n)
        n += x + gap
    qt = (torch.randn(n, heads, hd, generator=g) * sharp).to(D)
    return dict(q=qt, k_pages=kp, v_pages=vp, table=table, kv_len=torch.tensor(kv, dtype=torch.int32), q_start=torch.tensor(starts, dtype=torch.int32),
                q_len=torch.tensor(q, dtype=torch.int32), prefix_table=order[:npb].clone() if npb else None, prefix_len=prefix)


def run_case(pg, c, opts, out=None, **over):
    d = {k: (v.cuda() if hasattr(v, "cuda") else v) for k, v in c.items()}
    d.update(over)
    return pg.attention_dev(d["q"], d["k_pages"], d["v_pages"], d["table"], d["kv_len"], d["q_start"], d["q_len"],
                            max_q=over.get("max_q", max(1, int(c["q_len"].max()))), max_kv=over.get("max_kv", int(c["kv_len"].max())),
                            prefix_table=d["prefix_table"], prefix_len=d["prefix_len"], out=out, **opts)


def check_attention(pg, c, opts=None, **over):
    import torch
    opts = dict(opts or {})
    sent = torch.full(c["q"].shape, 7.0, dtype=c["q"].dtype)
    ocpu = {k: (v.cpu() if hasattr(v, "cpu") else v) for k, v in opts.items()}
    ref, tol = PO.attention(c["q"], c["k_pages"], c["v_pages"], c["table"], c["kv_len"], c["q_start"], c["q_len"], c["prefix_table"],
                            c["prefix_len"], out=sent, **ocpu)
    got = run_case(pg, c, opts, out=sent.cuda(), **over).cpu().double()
    err = (got - ref).abs()
    ok = err <= tol
    if not bool(ok.all()):
        bad = (~ok).nonzero()
        i = tuple(bad[0].tolist())
        raise AssertionError(f"{len(bad)} of {ok.numel()} off, first at {i}: {got[i]} for {ref[i]}, tol {tol[i]}; rows "
                             f"{sorted(set(bad[:, 0].tolist()))[:10]} heads {sorted(set(bad[:, 1].tolist()))[:10]}")
    return got


HEADS = [(32, 8, 128), (4, 4, 128), (8, 1, 64), (6, 2, 64), (14, 2, 128)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("heads,hk,hd", HEADS)
def test_decode(pg, dtype, heads, hk, hd):
    """One to a few tokens per request; lengths of one, page and tile borders, idle and ended requests."""
    kv = [1, 16, 17, 127, 128, 129, 255, 300, 40, 0, 64]
    q = [1, 1, 2, 1, 5, 1, 3, 1, 0, 0, 8]
    check_attention(pg, make_case(kv, q, heads, hk, hd, 16, dtype, seed=heads))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("prefix", [0, 1, 100, 256, 700])
def test_shared_prefix(pg, page, prefix):
    c = make_case([5, 1, 140, 33], [5, 1, 3, 2], 8, 2, 128, page, "bfloat16", prefix=prefix, seed=page + prefix)
    check_attention(pg, c)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,hk", [(8, 2), (6, 2), (2, 2)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_prompts(pg, heads, hk, hd, dtype):
    """Many new tokens per request: whole prompts, a chunk behind earlier positions, behind a prefix."""
    check_attention(pg, make_case([200, 333, 64], [200, 70, 64], heads, hk, hd, 16, dtype, seed=hd))
    check_attention(pg, make_case([130, 1, 300], [130, 1, 257], heads, hk, hd, 32, dtype, prefix=150, seed=hd + 1))


OPTS = [dict(softcap=5.0), dict(softcap=50.0), dict(alibi=True), dict(window=1), dict(window=20), dict(window=128), dict(window=150, softcap=3.0),
        dict(alibi=True, window=77, softcap=20.0), dict(scale=0.5), dict(scale=-0.1), dict(scale=0.0)]


@pytest.mark.parametrize("opts", OPTS, ids=lambda o: "-".join(f"{k}{v}" for k, v in o.items()))
@pytest.mark.parametrize("prefix", [0, 300])
def test_score_options(pg, opts, prefix):
    import torch
    opts = dict(opts)
    if opts.get("alibi"):
        opts["alibi"] = torch.exp2(-torch.arange(1, 9, dtype=torch.float32)).cuda()
    check_attention(pg, make_case([1, 100, 260, 31], [1, 4, 1, 31], 8, 2, 64, 16, "float16", prefix=prefix, seed=3), opts)
    check_attention(pg, make_case([300, 140], [300, 100], 8, 2, 128, 16, "bfloat16", prefix=prefix, seed=4), opts)


@pytest.mark.parametrize("opts", [dict()] + OPTS, ids=lambda o: "-".join(f"{k}{v}" for k, v in o.items()) or "plain")
@pytest.mark.parametrize("prefix", [0, 130])
@pytest.mark.parametrize("q,hd,dtype,page", [(1, 128, "bfloat16", 16), (2, 64, "float16", 32), (3, 128, "float16", 256), (4, 64, "bfloat16", 64)])
def test_few_rows(pg, q, hd, dtype, page, prefix, opts):
    """At most 16 rows per kv head (groups of 4 heads, up to 4 tokens): decode and short verifies, lengths around the
    borders of stages (64 keys), tiles and pages, idle and ended requests, several splits."""
    import torch
    opts = dict(opts)
    if opts.get("alibi"):
        opts["alibi"] = torch.exp2(-torch.arange(1, 9, dtype=torch.float32)).cuda()
    kv = [1, 63, 64, 65, 130, 0, 700, 17, 128, 1500]
    qs = [min(q, max(x, 1)) if i % 3 else min(1, x) for i, x in enumerate(kv)]
    qs[7] = 0
    check_attention(pg, make_case(kv, qs, 8, 2, hd, page, dtype, prefix=prefix, seed=q), opts)


@pytest.mark.parametrize("heads,hk,q", [(16, 1, 1), (17, 1, 1), (32, 1, 3), (100, 1, 2), (128, 1, 4), (65, 1, 3), (3, 3, 16), (3, 3, 17)])
def test_group_sizes(pg, heads, hk, q):
    """Groups from 1 to 128 heads per kv head, on both sides of 16 rows."""
    check_attention(pg, make_case([40, 200, 3], [q, min(q, 2), min(q, 3)], heads, hk, 64, 16, "bfloat16", prefix=20, seed=heads))


@pytest.mark.parametrize("q", [1, 9])
def test_no_keys_at_all(pg, q):
    """Every request empty: rows without a position are 0, and nothing is read."""
    for prefix in (0, 30):
        got = check_attention(pg, make_case([0, 0], [q, 1], 8, 2, 64, 16, "float16", prefix=prefix, seed=1), max_kv=0)
        assert not got.any()


@pytest.mark.parametrize("q", [2, 70])
def test_two_calls_at_once(pg, q):
    """Calls in flight on two streams, each again and again, give what each gives alone."""
    import torch
    cases = [make_case([300, 900, 40], [q, 1, 2], 8, 2, 128, 16, "bfloat16", prefix=200, seed=30 + i) for i in range(2)]
    dev = [{k: (v.cuda() if hasattr(v, "cuda") else v) for k, v in c.items()} for c in cases]

    def call(d):
        return pg.attention_dev(d["q"], d["k_pages"], d["v_pages"], d["table"], d["kv_len"], d["q_start"], d["q_len"], max_q=q,
                                max_kv=900, prefix_table=d["prefix_table"], prefix_len=200)
    want = [call(d) for d in dev]
    streams = [torch.cuda.Stream() for _ in dev]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(dev[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_one_query_for_all_tokens(pg):
    """q with a token stride of 0 (an expanded row)."""
    c = make_case([50, 90], [3, 1], 4, 2, 64, 16, "float16", seed=31)
    c["q"] = c["q"][:1].expand(4, -1, -1).clone()
    check_attention(pg, c, q=c["q"][:1].cuda().expand(4, -1, -1))


def test_rows_without_positions(pg):
    """More new tokens than positions: the first rows have no position and are 0; requests of length 0 too."""
    for prefix in (0, 40):
        got = check_attention(pg, make_case([3, 0, 2], [5, 2, 2], 8, 2, 128, 16, "float16", prefix=prefix, seed=9))
        assert not got[:2].any() and not got[5:7].any()


def test_padded_batch_is_left_alone(pg):
    """Rows between and behind the requests' tokens keep what out had (checked against the sentinel)."""
    check_attention(pg, make_case([40, 7, 200], [3, 0, 150], 8, 2, 128, 16, "bfloat16", prefix=33, seed=5, gap=4))
    check_attention(pg, make_case([40, 7, 200], [3, 1, 1], 8, 2, 64, 16, "float16", seed=5, gap=61))


@pytest.mark.parametrize("q", [1, 60])
@pytest.mark.parametrize("bad", [-1, -5, 1 << 30, "n_pages"])
def test_bad_pages_are_not_seen(pg, q, bad):
    c = make_case([70, 400, 64], [1, q, 2], 8, 2, 128, 16, "float16", prefix=48, seed=6)
    bad = c["k_pages"].shape[0] if bad == "n_pages" else bad
    c["table"][1, 3] = bad
    c["table"][1, 20:22] = bad
    c["prefix_table"][1] = bad
    check_attention(pg, c)
    assert error_word() == 3
    c["table"][2, :] = bad      # every page of a request, and the prefix: nothing to see
    c["prefix_table"][:] = bad
    check_attention(pg, c)
    assert error_word() == 3


def test_pages_outside_the_window_may_be_gone(pg):
    c = make_case([300, 420], [1, 4], 8, 2, 128, 16, "float16", prefix=64, seed=16)
    c["table"][0, :10] = -1
    c["table"][1, :18] = -1
    c["prefix_table"][:] = -1
    check_attention(pg, c, dict(window=100))
    error_word()  # whether such a page is recorded depends on the tiles


def test_lengths_past_the_bounds_are_cut(pg):
    import torch
    c = make_case([100, 50], [4, 2], 8, 2, 64, 16, "float16", seed=7)
    cut = dict(c, kv_len=torch.tensor([60, 50], dtype=torch.int32), q_len=torch.tensor([3, 2], dtype=torch.int32))
    sent = torch.full(c["q"].shape, 7.0, dtype=torch.float16)
    ref, tol = PO.attention(c["q"], c["k_pages"], c["v_pages"], c["table"], cut["kv_len"], c["q_start"], cut["q_len"], out=sent)
    got = run_case(pg, c, {}, out=sent.cuda(), max_q=3, max_kv=60).cpu().double()
    assert error_word() == 3
    assert bool(((got - ref).abs() <= tol).all())


@pytest.mark.parametrize("layout", ["hnd", "pair", "odd", "q_slice", "q_odd"])
@pytest.mark.parametrize("hd", [64, 128])
def test_strides(pg, layout, hd):
    import torch
    c = make_case([100, 300, 7], [1, 90, 7], 6, 2, hd, 16, "bfloat16", prefix=20, seed=8)
    n_pages, ps, hk, _ = c["k_pages"].shape
    over = {}
    if layout == "hnd":
        over = {k: c[k].transpose(1, 2).contiguous().cuda().transpose(1, 2) for k in ("k_pages", "v_pages")}
    elif layout == "pair":
        both = torch.stack([c["k_pages"], c["v_pages"]], 1).cuda()
        over = dict(k_pages=both[:, 0], v_pages=both[:, 1])
    elif layout == "odd":
        for k in ("k_pages", "v_pages"):
            w = torch.zeros(n_pages * ps * (hk * hd + 1) + 1, dtype=c[k].dtype, device="cuda")[1:].view(n_pages, ps, hk * hd + 1)
            w[..., :hk * hd] = c[k].flatten(2).cuda()
            over[k] = w[..., :hk * hd].unflatten(2, (hk, hd))
    else:
        pad = 8 if layout == "q_slice" else 3
        w = torch.zeros(c["q"].shape[0], c["q"].shape[1] + 1, hd + pad, dtype=c["q"].dtype, device="cuda")
        over["q"] = w[:, 1:, pad:]
        over["q"].copy_(c["q"])
    check_attention(pg, c, **over)


@pytest.mark.parametrize("hd", [8, 72, 96, 256])
def test_other_head_dims(pg, hd):
    check_attention(pg, make_case([40, 130], [3, 1], 6, 3, hd, 16, "float16", prefix=20, seed=hd))


def test_nan_in_a_row_stays_there(pg):
    """A query of NaN or infinity makes its own rows NaN only; its request's other rows and other requests are untouched."""
    import torch
    c = make_case([150, 60, 20], [40, 1, 3], 8, 2, 128, 16, "float16", prefix=30, seed=10)
    clean = run_case(pg, c, {}).cpu()
    c["q"][7, 2] = float("nan")
    c["q"][40, 5] = float("inf")
    got = run_case(pg, c, {}).cpu()
    assert torch.isnan(got[7, 2]).all() and not torch.isfinite(got[40, 5]).any()
    got[7, 2], got[40, 5] = clean[7, 2], clean[40, 5]
    assert torch.equal(got, clean)


def test_largest_scores(pg):
    """Scores near the type's largest values, all equal or one far above: softmax stays finite and exact."""
    import torch
    c = make_case([64, 200], [1, 80], 8, 2, 64, 16, "bfloat16", prefix=10, seed=11, sharp=300.0, poison=False)
    c["k_pages"] *= 40
    check_attention(pg, c)
    c["q"].fill_(0)
    check_attention(pg, c)


def test_same_bits_again_and_alone(pg):
    """The same call gives the same bits; a request's rows do not depend on what the others hold."""
    import torch
    c = make_case([500, 90, 1000, 3], [2, 1, 64, 1], 8, 2, 128, 16, "bfloat16", prefix=520, seed=12)
    a = run_case(pg, c, {})
    b = run_case(pg, c, {})
    assert torch.equal(a, b)
    d = dict(c, k_pages=c["k_pages"].clone(), v_pages=c["v_pages"].clone(), q=c["q"].clone())
    for r in (0, 1, 3):
        rows = d["table"][r][d["table"][r] >= 0].long()
        d["k_pages"][rows] = torch.randn_like(d["k_pages"][rows].float()).to(d["k_pages"].dtype)
        d["v_pages"][rows] = 1
    d["kv_len"] = torch.tensor([40, 1, 1000, 2], dtype=torch.int32)
    e = run_case(pg, d, {}, max_kv=1000)
    assert torch.equal(a[3:67], e[3:67])


def test_long_context(pg):
    """A context long enough for many splits, few rows; and a long prefix."""
    check_attention(pg, make_case([20000], [1], 8, 1, 64, 64, "float16", seed=13))
    check_attention(pg, make_case([5, 700], [1, 2], 4, 1, 128, 128, "bfloat16", prefix=9001, seed=14))


def test_many_requests(pg):
    rng = np.random.default_rng(15)
    n = 700
    kv = rng.integers(0, 60, n).tolist()
    q = [min(x, int(rng.integers(0, 4))) for x in kv]
    check_attention(pg, make_case(kv, q, 4, 2, 64, 16, "float16", prefix=50, seed=15))


def test_offsets_past_32_bits(pg):
    """Pages whose elements lie beyond 2^31 (and bytes beyond 2^32) in the pool."""
    import torch
    hk, hd, page = 8, 128, 256
    n_pages = (1 << 31) // (page * hk * hd) + 40
    c = make_case([600, 90], [2, 1], 32, hk, hd, page, "bfloat16", prefix=300, seed=17, spare=0, poison=False)
    big = {}
    used = c["k_pages"].shape[0]
    for k in ("k_pages", "v_pages"):
        big[k] = torch.empty(n_pages, page, hk, hd, dtype=torch.bfloat16, device="cuda")
        big[k][-used:] = c[k].cuda()
    shift = n_pages - used
    big["table"] = torch.where(c["table"] >= 0, c["table"] + shift, -1).cuda()
    big["prefix_table"] = (c["prefix_table"] + shift).cuda()
    check_attention(pg, c, **big)
    rows = torch.randn(3, hk, hd, device="cuda").bfloat16()
    slots = i32([n_pages * page - 1, (n_pages - 1) * page, (n_pages - used) * page + 7])
    pg.append_dev(rows, rows, slots, big["k_pages"], big["v_pages"])
    assert torch.equal(big["k_pages"].view(-1, hk, hd)[slots.long()], rows)


def test_other_stream_and_graph(pg):
    """On a side stream, and captured once and replayed with other lengths, tables and queries in place."""
    import torch
    c = make_case([90, 300, 20], [2, 40, 1], 8, 2, 128, 16, "float16", prefix=64, seed=18)
    want = run_case(pg, c, {})
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = run_case(pg, c, {})
    s.synchronize()
    assert torch.equal(want, got)
    d = {k: (v.cuda() if hasattr(v, "cuda") else v) for k, v in c.items()}
    out = torch.full_like(d["q"], 7.0)
    call = dict(max_q=40, max_kv=300, prefix_table=d["prefix_table"], prefix_len=64, out=out)
    args = (d["q"], d["k_pages"], d["v_pages"], d["table"], d["kv_len"], d["q_start"], d["q_len"])
    graphs = []
    for _ in range(2):  # two graphs of the same call, each with its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            pg.attention_dev(*args, **call)
        graphs.append(g)
    for kv, q in (([90, 300, 20], [2, 40, 1]), ([17, 200, 0], [1, 3, 0]), ([90, 250, 20], [0, 40, 1])):
        d["kv_len"].copy_(i32(kv))
        d["q_len"].copy_(i32(q))
        d["q"].normal_()
        for g in graphs:
            out.fill_(7.0)
            g.replay()
            torch.cuda.synchronize()
            ref, tol = PO.attention(d["q"].cpu(), c["k_pages"], c["v_pages"], c["table"], kv, c["q_start"], q, c["prefix_table"], 64,
                                    out=torch.full(c["q"].shape, 7.0))
            assert bool(((out.cpu().double() - ref).abs() <= tol).all())


# ---------------------------------------------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,opts", [("float16", {}), ("bfloat16", dict(softcap=20.0, window=90))])
def test_serving_steps(pg, dtype, opts):
    """A batch behind a shared prefix over several steps: prompts, verify steps with rejected drafts, requests that end
    and are replaced.  Pages from the plan, rows through the slot map, attention over them, against K and V kept as
    plain lists per request."""
    import torch
    D = getattr(torch, dtype)
    rng = np.random.default_rng(21)
    g = torch.Generator().manual_seed(21)
    B, hk, heads, hd, page, P, cap = 5, 2, 8, 64, 16, 45, 256
    pool = pg.PagePool(B + 1, 120, page, cap)
    kp = torch.full((120, page, hk, hd), float("nan"), dtype=D, device="cuda")
    vp = torch.full_like(kp, float("inf"))
    kept = [(torch.zeros(0, hk, hd, dtype=D), torch.zeros(0, hk, hd, dtype=D)) for _ in range(B)]
    prefix = tuple(torch.randn(P, hk, hd, generator=g).to(D) for _ in range(2))

    def step(kv, q, rows, n_tokens, pos0=0):
        plan = pool.plan(i32(kv), i32(q), n_tokens, pos0=pos0)
        assert plan.missing.item() == 0
        k, v = (torch.cat([r[i] for r in rows] + [torch.zeros(n_tokens - sum(len(r[i]) for r in rows), hk, hd, dtype=D)]) for i in (0, 1))
        pg.append_dev(k.cuda(), v.cuda(), plan.slots, kp, vp)
        return plan
    step([0] * B + [P], [0] * B + [P], [prefix], P + 3)  # the prefix is request B
    lens = [0] * B
    for it in range(8):
        q = []
        for b in range(B):
            if it == 0 or rng.random() < 0.15:
                lens[b], kept[b] = 0, (kept[b][0][:0], kept[b][1][:0])
                q.append(int(rng.integers(1, 120)))
            else:
                back = int(rng.integers(0, 4)) if lens[b] > 4 else 0  # rejected drafts of the last step
                lens[b] -= back
                kept[b] = tuple(x[:lens[b]] for x in kept[b])
                q.append(min(int(rng.integers(0, 6)), cap - lens[b]))
        rows = [tuple(torch.randn(n, hk, hd, generator=g).to(D) for _ in range(2)) for n in q]
        lens = [a + b for a, b in zip(lens, q)]
        kept = [tuple(torch.cat([x, y]) for x, y in zip(kept[b], rows[b])) for b in range(B)]
        n_tokens = sum(q) + 2
        plan = step(lens + [P], q + [0], rows, n_tokens, pos0=P)
        qt = torch.randn(n_tokens, heads, hd, generator=g).to(D)
        out = torch.full((n_tokens, heads, hd), 7.0, dtype=D, device="cuda")
        pg.attention_dev(qt.cuda(), kp, vp, pool.table[:B], i32(lens), plan.q_start[:B], i32(q), max_q=max(q), max_kv=max(lens),
                         prefix_table=pool.table[B], prefix_len=P, out=out, **opts)
        # the same in plain pages: request b's keys in one page of its own
        ks = torch.zeros(B + 1, cap, hk, hd, dtype=D)
        vs = torch.zeros_like(ks)
        for b in range(B):
            ks[b, :lens[b]], vs[b, :lens[b]] = kept[b]
        ks[B, :P], vs[B, :P] = prefix
        ref, tol = PO.attention(qt, ks, vs, torch.arange(B, dtype=torch.int32)[:, None], lens, plan.q_start[:B].tolist(), q,
                                torch.tensor([B], dtype=torch.int32), P, out=torch.full(qt.shape, 7.0), **opts)
        assert bool(((out.cpu().double() - ref).abs() <= tol).all()), it
