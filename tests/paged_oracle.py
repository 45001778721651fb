"""Plain 64-bit restatements of the paged K/V cache operators, for the tests (numpy / torch on the CPU).

Attention also returns how far an fp32-accumulating kernel may be off, element by element.  With e the half step of
the pool's type relative to the value (torch.finfo(t).eps / 2):
  - the output is rounded once: e |o|;
  - the weights p are rounded once before the product with V: e sum p |v|, where p sums to 1; an fp16 weight below the
    type's normal range is off by at most 2^-25 in units where the largest weight is at least 2^6: n 2^-31 max |v|;
  - a score z is off by dz <= scale (d + 8) 2^-22 max_j sum |q k_j| (an fp32 dot product of d terms, adds that may
    truncate), 2^-21 |z|max (its fp32 scaling and the base change of exp), softcap 2^-21 and slope * distance 2^-22:
    each weight by a factor within exp(+-dz), the output by 2 dz sum p |v|;
  - exp2 (2^-22 relative) and the fp32 sums over n keys in any order (n 2^-23, at most 2^-12): 2^-12 sum p |v| at most.
    The sums run over tiles and splits, so 2^-16 covers the lengths used here (partial sums of at most 2^7 terms each
    pass 2^-16 / 2^-23 = 2^7 roundings).
"""
import math

import torch

EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def plan(state, kv_len, q_len, page, n_tokens, q_stride=0, pos0=0):
    """state: dict(table list of lists, free list, ld).  Mutates it; returns q_start, slots, positions, missing."""
    table, free, ld = state["table"], state["free"], state["ld"]
    need = [-(-min(max(k, 0), ld * page) // page) for k in kv_len]
    for b, row in enumerate(table):
        while_from = need[b]
        free.extend(row[while_from:])
        del row[while_from:]
    missing = 0
    for b, row in enumerate(table):
        while len(row) < need[b]:
            if not free:
                missing += need[b] - len(row)
                break
            row.append(free.pop())
    q_start, slots, positions, at = [], [-1] * n_tokens, [-1] * n_tokens, 0
    for b, (k, q) in enumerate(zip(kv_len, q_len)):
        start = b * q_stride if q_stride else at
        q_start.append(start)
        at += q
        for t in range(q):
            p = k - q + t
            if start + t >= n_tokens or p < 0:
                continue
            positions[start + t] = pos0 + p
            if p // page < len(table[b]):
                slots[start + t] = table[b][p // page] * page + p % page
    return q_start, slots, positions, missing


def attention(q, k_pages, v_pages, table, kv_len, q_start, q_len, prefix_table=None, prefix_len=0, scale=None, softcap=0.0,
              window=0, alibi=None, out=None):
    """CPU tensors; returns (out, tol) in float64.  Positions whose page is outside the pool are not seen."""
    n_tok, H, D = q.shape
    n_pages, ps, hk, _ = k_pages.shape
    G = H // hk
    e = EPS[q.dtype]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    ref = out.double().clone() if out is not None else torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros_like(ref)
    for b in range(len(kv_len)):
        L, T, s0 = int(kv_len[b]), int(q_len[b]), int(q_start[b])
        if T <= 0:
            continue
        pos = torch.arange(prefix_len + L)
        pages = torch.cat([prefix_table.long()[torch.arange(prefix_len) // ps] if prefix_len else torch.zeros(0, dtype=torch.long),
                           table[b].long()[torch.arange(L) // ps]])
        off = torch.cat([torch.arange(prefix_len) % ps, torch.arange(L) % ps])
        there = (pages >= 0) & (pages < n_pages)
        K = torch.zeros(len(pos), hk, D, dtype=torch.float64)
        V = torch.zeros_like(K)
        K[there] = k_pages[pages[there], off[there]].double()
        V[there] = v_pages[pages[there], off[there]].double()
        for t in range(T):
            i = L - T + t
            me = prefix_len + i
            seen = there & (pos <= me)
            if window:
                seen &= me - pos < window
            row = s0 + t
            ref[row] = 0.0
            if i < 0 or not bool(seen.any()):
                continue
            qs = q[row].double().view(hk, G, 1, D)
            Ks, Vs, dist = K[seen].transpose(0, 1), V[seen].transpose(0, 1), (me - pos[seen]).double()  # [hk, n, D]
            z = (qs * Ks[:, None]).sum(-1) * scale  # [hk, G, n]
            zmax = z.abs().amax(-1, keepdim=True)
            mag = (qs.abs() * Ks[:, None].abs()).sum(-1).amax(-1, keepdim=True) * abs(scale)
            dz = mag * (D + 8) * 2.0 ** -22 + zmax * 2.0 ** -21
            if softcap:
                z = softcap * torch.tanh(z / softcap)
                dz = dz + softcap * 2.0 ** -21
            if alibi is not None:
                sl = alibi.double().view(hk, G, 1)
                z = z - sl * dist
                dz = dz + sl.abs() * dist.max() * 2.0 ** -22
            p = torch.softmax(z, -1)
            o = torch.einsum("hgn,hnd->hgd", p, Vs)
            pv = torch.einsum("hgn,hnd->hgd", p, Vs.abs())
            n = dist.numel()
            # |o| (1 + small) e + e pv: the weights' and the output's rounding, and the terms above
            err = e * pv + (2 * dz + 2.0 ** -16) * pv + n * 2.0 ** -31 * Vs.abs().amax(1)[:, None]
            ref[row] = o.reshape(H, D)
            tol[row] = (err + e * (o.abs() + err)).reshape(H, D) + 2.0 ** -24
    return ref, tol
