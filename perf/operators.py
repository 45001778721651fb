"""The paged K/V cache of batched serving, as it is measured: block tables and slot maps built from request lengths,
K/V rows written through the slot map, and attention over the pages (a batch that shares a long prefix; scores
capped by a tanh or biased by distance; windows; prompts packed one after another).

``run`` computes each operator in its plain form with elementary torch operations, or, where ``own`` is true, makes
the calls a user makes of anetransformers_b200.paged.

Pages.  A pool has n_pages pages of page_size positions.  Request b holds held[b] pages, named in order by its row of
the block table (-1 behind them); the free pages are a stack (free[0 .. n_free), -1 above it).  One plan takes the
lengths after this step (kv_len, q_len new positions at the end): requests that shrank give their last pages back
(pushed in ascending (request, page) order), then requests that grew take pages from the top of the stack in ascending
(request, page) order; where the stack is empty the entry stays -1 and is counted as missing.  New token t of request
b sits at position p = kv_len[b] - q_len[b] + t, slot table[b][p // page_size] * page_size + p % page_size.

Attention.  Row t of request b sees the shared prefix (positions 0 .. prefix_len - 1) and its request's own positions
0 .. kv_len - q_len + t, which follow the prefix.  score = scale * q.k, then cap * tanh(score / cap) (softcap), then
- slope[head] * distance (alibi); only distances below window are seen (window).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one stream that decodes: the smallest step, all latency
        dict(name="pages_one", op="pages", n_req=1, page=16, max_len=4096, q=1, prompts=False, fill=1.1),
        # a verify step of many streams: 5 tokens each, a tenth of the streams finished and replaced
        dict(name="pages_verify", op="pages", n_req=256, page=16, max_len=32768, q=5, prompts=False, fill=1.1),
        # a wave of ragged prompts that replaces another
        dict(name="pages_prompts", op="pages", n_req=64, page=64, max_len=2048, q=1024, prompts=True, fill=1.1),
        # K/V of a verify step: 64 streams x 5 tokens, cut out of the rows of a 6144-wide fp32 QKV product
        dict(name="append_verify", op="append", n_req=64, q=5, kv_heads=8, head_dim=128, page=16, src="f32", dtype="f16"),
        # K/V of a wave of prompts
        dict(name="append_prompts", op="append", n_req=16, q=1024, kv_heads=8, head_dim=128, page=64, src="bf16", dtype="bf16"),
        # one stream, one token, a short context: latency
        dict(name="attn_one", op="attn", n_req=1, q_min=1, q_max=1, prefix=0, own_min=128, own_max=128, heads=32, kv_heads=8,
             head_dim=128, page=16, dtype="f16", cap=0.0, alibi=False, window=0),
        # verify step of 64 streams x 5 tokens behind one 4096-token prefix, short contexts of their own
        dict(name="shared_verify", op="attn", n_req=64, q_min=5, q_max=5, prefix=4096, own_min=16, own_max=512, heads=32,
             kv_heads=8, head_dim=128, page=16, dtype="f16", cap=0.0, alibi=False, window=0),
        # decode of 32 streams behind a document of 32768 tokens
        dict(name="shared_long", op="attn", n_req=32, q_min=1, q_max=1, prefix=32768, own_min=1, own_max=1024, heads=32,
             kv_heads=8, head_dim=128, page=64, dtype="bf16", cap=0.0, alibi=False, window=0),
        # prompts of 8 requests behind a shared prefix
        dict(name="shared_prompts", op="attn", n_req=8, q_min=100, q_max=1024, prefix=8192, own_min=100, own_max=1024, heads=32,
             kv_heads=8, head_dim=128, page=32, dtype="bf16", cap=0.0, alibi=False, window=0),
        # decode of 64 streams with ragged contexts up to 8192, capped scores
        dict(name="capped_decode", op="attn", n_req=64, q_min=1, q_max=1, prefix=0, own_min=1, own_max=8192, heads=32, kv_heads=8,
             head_dim=128, page=16, dtype="bf16", cap=30.0, alibi=False, window=0),
        # four ragged prompts packed one after another, capped scores
        dict(name="capped_prompts", op="attn", n_req=4, q_min=301, q_max=4096, prefix=0, own_min=301, own_max=4096, heads=32,
             kv_heads=8, head_dim=128, page=16, dtype="bf16", cap=50.0, alibi=False, window=0),
        # two chunks of long prompts over contexts of up to 16384, distance bias and a window, narrow heads
        dict(name="biased_prompts", op="attn", n_req=2, q_min=2000, q_max=2048, prefix=0, own_min=5001, own_max=16384, heads=32,
             kv_heads=8, head_dim=64, page=32, dtype="f16", cap=0.0, alibi=True, window=4096),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6e12 + w["flops"] / 1e15


def draw(rng):
    op = rng.choice(["pages", "append", "attn", "attn", "attn"])
    if op == "pages":
        prompts = rng.random() < 0.4
        n_req = _log(rng, 1, 256 if not prompts else 64)
        q = _log(rng, 2, 65536 // n_req // 2) if prompts else rng.randint(1, 16)
        if prompts:
            q = min(q, 8192)
        return dict(op=op, n_req=n_req, page=rng.choice([16, 32, 64, 128, 256]), max_len=2 * q if prompts else _log(rng, 64, 32768),
                    q=q, prompts=prompts, fill=rng.choice([1.1, 1.1, 0.9]))
    if op == "append":
        n_req = _log(rng, 1, 64)
        dtype = rng.choice(["f16", "bf16"])
        return dict(op=op, n_req=n_req, q=_log(rng, 1, 16384 // n_req), kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128]),
                    page=rng.choice([16, 32, 64, 128, 256]), src=rng.choice(["f32", dtype]), dtype=dtype)
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (32, 32), (16, 2), (12, 4), (14, 2), (8, 1), (20, 4)])
    shape = rng.choice(["decode", "shared", "prompts"])
    c = dict(op=op, n_req=_log(rng, 1, 64), q_min=1, q_max=rng.randint(1, 8), prefix=0, own_min=1, own_max=_log(rng, 16, 8192), heads=heads,
             kv_heads=kv_heads, head_dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128, 256]), dtype=rng.choice(["f16", "bf16"]),
             cap=rng.choice([0.0, 0.0, 15.0, 50.0]), alibi=rng.random() < 0.25, window=rng.choice([0, 0, 0, _log(rng, 16, 8192)]))
    if shape == "shared":
        c.update(prefix=_log(rng, 100, 32768), own_max=_log(rng, 16, 2048))
    elif shape == "prompts":
        c.update(n_req=_log(rng, 1, 8), q_max=_log(rng, 32, 4096), prefix=rng.choice([0, 0, _log(rng, 100, 8192)]))
        c.update(q_min=max(1, c["q_max"] // rng.randint(1, 16)))
    c["own_max"] = max(c["own_max"], c["q_max"])
    c["own_min"] = max(1, c["q_min"], c["own_max"] // rng.choice([1, 4, 64, 10000]))
    most = max(_cost(x) for x in listed())
    while _cost(c) > most:
        for k in ("n_req", "prefix", "own_max", "q_max"):
            c[k] = c[k] * 3 // 4 if k == "prefix" else max(1, c[k] * 3 // 4)
        c["q_min"] = min(c["q_min"], c["q_max"])
        c["own_max"] = max(c["own_max"], c["q_max"])
        c["own_min"] = max(1, c["q_min"], min(c["own_min"], c["own_max"]))
    return c


def _spread(lo, hi, n, salt):
    """n lengths from lo to hi, evenly over the range, in an order that depends on the sizes only."""
    v = [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    return [v[i] for i in np.random.RandomState(salt + n).permutation(n)]


def _lengths(case):
    """(kv_len, q_len) of the attention requests."""
    kv = _spread(case["own_min"], case["own_max"], case["n_req"], 11)
    q = _spread(case["q_min"], case["q_max"], case["n_req"], 12)
    return kv, [min(a, b) for a, b in zip(q, kv)]


def _page_lengths(case):
    """Two (kv_len, q_len) pairs: consecutive steps of a serving loop."""
    n, r = case["n_req"], np.random.RandomState(case["n_req"] + case["max_len"])
    if case["prompts"]:
        a = _spread(max(1, case["q"] // 8), case["q"], n, 13)
        b = _spread(max(1, case["q"] // 16), case["q"], n, 14)
        return (a, a), (b, b)
    q = min(case["q"], case["max_len"])
    a = [min(case["max_len"], x + q) for x in _spread(1, max(1, case["max_len"] - 2 * q), n, 15)]
    b = [min(case["max_len"], x + int(r.randint(1, q + 1))) if r.rand() < 0.9 else q + int(r.randint(0, case["max_len"] - q + 1)) for x in a]
    return (a, [q] * n), (b, [q] * n)


def work(case):
    if case["op"] == "pages":
        n, ps = case["n_req"], case["page"]
        steps = _page_lengths(case)
        tokens = sum(sum(q) for _, q in steps) / 2
        moved = sum(abs(-(-x // ps) - -(-y // ps)) for x, y in zip(steps[0][0], steps[1][0]))
        return {"bytes": 4 * (5 * n + 2 * tokens + 4 * moved + 4), "flops": 0}
    if case["op"] == "append":
        n = case["n_req"] * case["q"]
        row = case["kv_heads"] * case["head_dim"]
        return {"bytes": 2 * n * row * (2 + (4 if case["src"] == "f32" else 2)) + 4 * n, "flops": 0}
    kv, q = _lengths(case)
    hd, P, W = case["head_dim"], case["prefix"], case["window"]
    seen = rows = own_keys = prefix_keys = 0
    for L, T in zip(kv, q):
        rows += T
        first = P + L - T  # keys before the first row's own
        if not W:
            seen += T * (first + 1) + T * (T - 1) // 2
            own_keys += L
            prefix_keys = P
        else:
            seen += sum(min(first + t + 1, W) for t in range(T))
            own_keys += min(L, T + W - 1)
            prefix_keys = max(prefix_keys, min(P, max(0, W - 1 - (L - T))))
    return {"bytes": 2 * (2 * rows * case["heads"] * hd + 2 * (own_keys + prefix_keys) * case["kv_heads"] * hd),
            "flops": 4 * hd * case["heads"] * seen}


def _rand(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _rand(seed)
    st = dict(case)
    if own:
        from anetransformers_b200 import paged
        st["api"] = paged
    if case["op"] == "pages":
        steps = _page_lengths(case)
        ps, n = case["page"], case["n_req"]
        need = max(sum(-(-x // ps) for x in kv) for kv, _ in steps)
        n_pages = max(1, int(need * case["fill"]))
        # inputs of another seed: the requests in another order, and a free stack as a pool in use has it
        order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist()
        st["steps"] = [(_i32([kv[i] for i in order]), _i32([q[i] for i in order])) for kv, q in steps]
        st["n_tokens"] = max(sum(q) for _, q in steps)
        st["n_pages"], st["at"] = n_pages, 0
        free = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        if own:
            st["pool"] = paged.PagePool(n, n_pages, ps, case["max_len"])
            st["pool"].free.copy_(free)
        else:
            st["table"] = torch.full((n, -(-case["max_len"] // ps)), -1, dtype=torch.int32, device="cuda")
            st["held"] = torch.zeros(n, dtype=torch.int32, device="cuda")
            st["free"] = free
            st["n_free"] = torch.full((1,), n_pages, dtype=torch.int32, device="cuda")
        return st
    hd, hk, ps = case["head_dim"], case["kv_heads"], case["page"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "append":
        n = case["n_req"] * case["q"]
        per = -(-case["q"] // ps) + 1
        pages = torch.randperm(case["n_req"] * per, generator=g, device="cuda").view(case["n_req"], per)
        pos = torch.arange(case["q"], device="cuda") + ps // 2  # requests whose step starts in the middle of a page
        st["slots"] = (pages[:, pos // ps] * ps + pos % ps).reshape(-1).to(torch.int32)
        wide = torch.randn(n, 6 * hk * hd, generator=g, device="cuda").to(DTYPES[case["src"]])
        st["k"] = wide[:, 4 * hk * hd:5 * hk * hd].unflatten(1, (hk, hd))
        st["v"] = wide[:, 5 * hk * hd:].unflatten(1, (hk, hd))
        st["k_pool"] = torch.zeros(case["n_req"] * per, ps, hk, hd, dtype=dt, device="cuda")
        st["v_pool"] = torch.zeros_like(st["k_pool"])
        return st
    kv, q = _lengths(case)
    blocks = [-(-x // ps) for x in kv]
    prefix_blocks = -(-case["prefix"] // ps)
    n_pages = sum(blocks) + prefix_blocks
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    st["prefix_table"] = order[:prefix_blocks].contiguous() if prefix_blocks else None
    table = torch.full((case["n_req"], max(blocks)), -1, dtype=torch.int32, device="cuda")
    at = prefix_blocks
    for b, m in enumerate(blocks):
        table[b, :m] = order[at:at + m]
        at += m
    st["table"] = table
    st["k_pool"] = torch.randn(n_pages, ps, hk, hd, generator=g, device="cuda", dtype=dt)
    st["v_pool"] = torch.randn(n_pages, ps, hk, hd, generator=g, device="cuda", dtype=dt) + torch.randn(hk, hd, generator=g, device="cuda").to(dt) * 0.25
    # scores of about 2 in standard deviation: a few keys carry most of a row's weight
    st["q"] = (torch.randn(sum(q), case["heads"], hd, generator=g, device="cuda") * 2).to(dt)
    st["kv_list"], st["q_list"] = kv, q
    st["kv_len"], st["q_len"] = _i32(kv), _i32(q)
    st["q_start"] = _i32([sum(q[:b]) for b in range(case["n_req"])])
    st["scale"] = 1.0 / math.sqrt(hd)
    st["slopes"] = None
    if case["alibi"]:
        h = torch.arange(1, case["heads"] + 1, device="cuda", dtype=torch.float32)
        st["slopes"] = torch.exp2(-8.0 * h / case["heads"])
    return st


# ---------------------------------------------------------------------------------------------------------------
# The calls of a user's program
# ---------------------------------------------------------------------------------------------------------------
def run(st):
    if st["op"] == "pages":
        kv_len, q_len = st["steps"][st["at"]]
        st["at"] ^= 1
        return _pages_own(st, kv_len, q_len) if own else _pages_plain(st, kv_len, q_len)
    if st["op"] == "append":
        if own:
            st["api"].append_dev(st["k"], st["v"], st["slots"], st["k_pool"], st["v_pool"])
        else:
            _append_plain(st)
        return st["k_pool"], st["v_pool"]
    return _attn_own(st) if own else _attn_plain(st)


def _pages_own(st, kv_len, q_len):
    pool = st["pool"]
    p = pool.plan(kv_len, q_len, st["n_tokens"])
    return dict(table=pool.table, held=pool.held, free=pool.free, n_free=pool.n_free, q_start=p.q_start, slots=p.slots,
                positions=p.positions, missing=p.missing)


def _attn_own(st):
    return st["api"].attention_dev(st["q"], st["k_pool"], st["v_pool"], st["table"], st["kv_len"], st["q_start"], st["q_len"],
                                   max_q=max(st["q_list"]), max_kv=max(st["kv_list"]), prefix_table=st["prefix_table"],
                                   prefix_len=st["prefix"], scale=st["scale"], softcap=st["cap"], window=st["window"],
                                   alibi=st["slopes"])


# ---------------------------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------------------------
def _pages_plain(st, kv_len, q_len):
    ps, table, held, free, n_free = st["page"], st["table"], st["held"], st["free"], st["n_free"]
    n, ld = table.shape
    dev = table.device
    idx = torch.arange(ld, device=dev)
    need = ((kv_len.long() + ps - 1) // ps)[:, None]
    had = held.long()[:, None]
    count = n_free.long()
    # pages given back, pushed in ascending order
    back = (idx >= need) & (idx < had)
    rank = torch.cumsum(back.reshape(-1).long(), 0).view(n, ld) - 1
    n_back = back.sum()
    spare = torch.cat([free, free.new_full((1,), -1)])
    spare.index_copy_(0, torch.where(back, count + rank, st["n_pages"]).reshape(-1).clamp_(max=st["n_pages"]), table.reshape(-1))
    new_free = spare[:st["n_pages"]]
    count = count + n_back
    # pages taken, from the top
    want = (idx >= had) & (idx < need)
    rank = torch.cumsum(want.reshape(-1).long(), 0).view(n, ld) - 1
    n_want = want.sum()
    got = want & (rank < count)
    taken = new_free[(count - 1 - rank).clamp(0, st["n_pages"] - 1)]
    new_table = torch.where(back, -1, torch.where(got, taken, table)).to(torch.int32)
    missing = (n_want - count).clamp(min=0)
    count = (count - n_want).clamp(min=0)
    table.copy_(new_table)
    held.copy_((table >= 0).sum(1))
    free.copy_(torch.where(torch.arange(st["n_pages"], device=dev) < count, new_free, -1))
    n_free.copy_(count)
    # tokens
    ends = torch.cumsum(q_len.long(), 0)
    q_start = (ends - q_len).to(torch.int32)
    tok = torch.arange(st["n_tokens"], device=dev)
    b = torch.searchsorted(ends, tok, right=True)
    live = b < n
    b = b.clamp(max=n - 1)
    pos = kv_len[b].long() - q_len[b] + tok - q_start[b]
    page = table[b, (pos // ps).clamp(0, ld - 1)].long()
    ok = live & (page >= 0) & (pos >= 0)
    slots = torch.where(ok, page * ps + pos % ps, -1).to(torch.int32)
    positions = torch.where(live, pos, -1).to(torch.int32)
    return dict(table=table, held=held, free=free, n_free=n_free, q_start=q_start, slots=slots, positions=positions,
                missing=missing.to(torch.int32).reshape(1))


def _append_plain(st):
    for src, pool in ((st["k"], st["k_pool"]), (st["v"], st["v_pool"])):
        pool.view(-1, *pool.shape[2:])[st["slots"].long()] = src.to(pool.dtype)


def _rows(pool, table, n):
    """The first n positions of a request (or the prefix) as [n, heads, dim]."""
    return pool[table[:-(-n // pool.shape[1])].long()].flatten(0, 1)[:n]


def _attn_plain(st):
    out = torch.empty_like(st["q"])
    G, P, W = st["heads"] // st["kv_heads"], st["prefix"], st["window"]
    kp = vp = None
    if P:
        kp, vp = _rows(st["k_pool"], st["prefix_table"], P).float(), _rows(st["v_pool"], st["prefix_table"], P).float()
    at = 0
    for b, (L, T) in enumerate(zip(st["kv_list"], st["q_list"])):
        k, v = _rows(st["k_pool"], st["table"][b], L).float(), _rows(st["v_pool"], st["table"][b], L).float()
        if P:
            k, v = torch.cat([kp, k]), torch.cat([vp, v])
        k, v = k.permute(1, 2, 0), v.permute(1, 0, 2)  # [kv_heads, dim, n], [kv_heads, n, dim]
        step = max(1, min(T, (1 << 28) // (st["heads"] * (P + L))))
        for t0 in range(0, T, step):
            t1 = min(T, t0 + step)
            q = st["q"][at + t0:at + t1].float().unflatten(1, (-1, G)).permute(1, 2, 0, 3)  # [kv_heads, G, t, dim]
            s = (q.flatten(1, 2) @ k).unflatten(1, (G, t1 - t0)) * st["scale"]
            if st["cap"]:
                s = st["cap"] * torch.tanh(s / st["cap"])
            dist = (P + L - T + torch.arange(t0, t1, device=s.device))[:, None] - torch.arange(P + L, device=s.device)
            if st["slopes"] is not None:
                s = s - st["slopes"].view(-1, G, 1, 1) * dist.float()
            hidden = dist < 0
            if W:
                hidden = hidden | (dist >= W)
            s = s.masked_fill(hidden, float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            o = (p.flatten(1, 2) @ v).unflatten(1, (G, t1 - t0)) / p.sum(-1, keepdim=True)
            out[at + t0:at + t1] = o.permute(2, 0, 1, 3).flatten(1, 2).to(out.dtype)
        at += T
    return out


# ---------------------------------------------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "pages":
        return None  # whole numbers
    st = prepare(case, seed)
    if case["op"] == "append":
        pools = []
        where = st["slots"].cpu().numpy()
        for src, pool in ((st["k"], st["k_pool"]), (st["v"], st["v_pool"])):
            flat = np.zeros((pool.shape[0] * pool.shape[1], pool.shape[2] * pool.shape[3]))
            flat[where] = src.double().cpu().numpy().reshape(len(where), -1)
            pools.append(torch.from_numpy(flat.reshape(tuple(pool.shape))))
        return tuple(pools)
    ps, P, W, cap = case["page"], case["prefix"], case["window"], case["cap"]
    G, dev = case["heads"] // case["kv_heads"], st["q"].device
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=dev)
    for b in range(case["n_req"]):
        L, T, first = st["kv_list"][b], st["q_list"][b], int(st["q_start"][b])
        # the pool row of every key that the request can see, by its position
        place = torch.arange(L, device=dev)
        place = st["table"][b].long()[place // ps] * ps + place % ps
        if P:
            head = torch.arange(P, device=dev)
            place = torch.cat([st["prefix_table"].long()[head // ps] * ps + head % ps, place])
        key_pos = torch.arange(P + L, dtype=torch.float64, device=dev)
        for h in range(case["heads"]):
            K = st["k_pool"].flatten(0, 1)[place, h // G].double()
            V = st["v_pool"].flatten(0, 1)[place, h // G].double()
            for t0 in range(0, T, 2048):
                Q = st["q"][first + t0:first + min(T, t0 + 2048), h].double()
                row_pos = P + L - T + t0 + torch.arange(len(Q), dtype=torch.float64, device=dev)
                z = torch.einsum("td,nd->tn", Q, K) * st["scale"]
                if cap:
                    z = torch.tanh(z / cap) * cap
                away = row_pos.unsqueeze(1) - key_pos.unsqueeze(0)
                if st["slopes"] is not None:
                    z -= away * float(st["slopes"][h])
                seen = (away >= 0) & (away < (W or float("inf")))
                z = torch.where(seen, z, torch.full_like(z, -float("inf")))
                weight = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
                out[first + t0:first + t0 + len(Q), h] = torch.einsum("tn,nd->td", weight, V)
    return out
