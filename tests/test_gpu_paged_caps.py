"""Capped scores of the paged attention over the whole range of caps that it takes, in each of its kernels.

The bound of tests/paged_oracle.py grants an absolute error of softcap * 2^-21 per score, which at a cap of 1e6 is half a
unit.  Here the cap's error is relative to the capped score z = c tanh(x):
  - |x| <= 1/2: x times a polynomial in x^2, 6.4e-7 relative, and its roundings (multiplications and fused adds whose
    terms after the first are at most x^2 / 3 of it): within 2^-20;
  - |x| > 1/2: c (1 - r) with r = 2 / (1 + E), E = e^(2x).  E is off by 2^-22 (ex2) and 6 |x| 2^-24 (three roundings of its
    argument, times the slope) relative, which moves r by r E / (1 + E) = 2 E / (1 + E)^2 <= 0.394 times that, so by at most
    0.394 * 7 * 2^-24 = 2.8 * 2^-24 at |x| = 1/2 (it falls from there); the reciprocal adds r 2^-23 <= 2.93 * 2^-24, the last
    rounding 2^-24: 6.8 * 2^-24 c against |z| >= 0.462 c, 14.6 * 2^-24 relative, and the constants' roundings one more:
    within 2^-20.
The other terms are those of tests/paged_oracle.py.
"""
import math

import pytest

from tests import paged_oracle as PO
from tests.conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs a CUDA GPU")]


def capped(q, k, v, kv_len, q_len, scale, cap):
    """One request after another, keys k, v [request][n][kv heads][D]; (out, bound) in 64 bits."""
    import torch
    e = PO.EPS[q.dtype]
    D, hk = q.shape[2], k[0].shape[1]
    out, tol, row = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), 0
    for K, V, L, T in zip(k, v, kv_len, q_len):
        for t in range(T):
            n = L - T + t + 1
            Ks, Vs = K[:n].double().transpose(0, 1), V[:n].double().transpose(0, 1)
            qs = q[row].double().view(hk, -1, 1, D)
            s = (qs * Ks[:, None]).sum(-1) * scale
            z = cap * torch.tanh(s / cap)
            mag = (qs.abs() * Ks[:, None].abs()).sum(-1).amax(-1, keepdim=True) * abs(scale)
            dz = mag * (D + 8) * 2.0 ** -22 + s.abs().amax(-1, keepdim=True) * 2.0 ** -21 + z.abs().amax(-1, keepdim=True) * 2.0 ** -20
            p = torch.softmax(z, -1)
            o, pv = torch.einsum("hgn,hnd->hgd", p, Vs), torch.einsum("hgn,hnd->hgd", p, Vs.abs())
            err = e * pv + (2 * dz + 2.0 ** -16) * pv + n * 2.0 ** -31 * Vs.abs().amax(1)[:, None]
            out[row] = o.flatten(0, 1)
            tol[row] = (err + e * (o.abs() + err)).flatten(0, 1) + 2.0 ** -24
            row += 1
    return out, tol


def check(kv_len, q_len, heads, hk, hd, dtype, cap, scale=None, size=1.0, page=16):
    import torch
    from anetransformers_b200 import paged
    g = torch.Generator().manual_seed(hd + sum(q_len))
    D = getattr(torch, dtype)
    n = max(-(-x // page) for x in kv_len)
    kp, vp = (torch.randn(len(kv_len) * n, page, hk, hd, generator=g) for _ in range(2))
    kp, vp = (kp * size).to(D), vp.to(D)
    table = torch.randperm(len(kv_len) * n, generator=g).to(torch.int32).view(len(kv_len), n)
    q = (torch.randn(sum(q_len), heads, hd, generator=g) * 2 * size).to(D)
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    got = paged.attention_dev(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), i32(kv_len), i32([sum(q_len[:b]) for b in range(len(q_len))]),
                              i32(q_len), max_q=max(q_len), max_kv=max(kv_len), scale=scale, softcap=cap).cpu().double()
    rows = [[x[table[b].long()].flatten(0, 1) for b in range(len(kv_len))] for x in (kp, vp)]
    ref, tol = capped(q, *rows, kv_len, q_len, scale, cap)
    err = (got - ref).abs()
    assert bool((err <= tol).all()), f"{float((err / tol).max()):.1f} times the bound"


# requests of one to four tokens (few rows per kv head), of up to 70 (tiles of 128 rows), and a head size without either
@pytest.mark.parametrize("q_len,hd", [([1, 1, 1], 128), ([1, 3, 2], 64), ([2, 70, 40], 128), ([2, 70, 40], 64), ([1, 3, 2], 72)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("cap", [1e-6, 0.25, 1.0, 5.0, 50.0, 1e4, 1e6, 1e9, 1e30])
def test_caps(cap, dtype, q_len, hd):
    check([512, 300, 77], q_len, 8, 2, hd, dtype, cap)


@pytest.mark.parametrize("q_len", [[1, 2], [90, 2]])
@pytest.mark.parametrize("scale,cap", [(1e-20, 1e30), (1e-20, 30.0), (-1e-20, 1e30), (1e-20, 1e4)])
def test_small_scales(scale, cap, q_len):
    """Scores of a few units from products of 1e20: scale / cap itself may lie below what 32 bits hold."""
    check([200, 150], q_len, 8, 2, 64, "bfloat16", cap, scale=scale, size=3e9)
