"""Attention over a shared prefix from its definition, in 64 bits on the CPU."""

import math

import torch


def rotate(x, cs):
    """NeoX halves of x [.., heads, 128] at cs [.., 128] = cos | sin."""
    a, b = x[..., :64].double(), x[..., 64:].double()
    c, s = cs[..., None, :64].double(), cs[..., None, 64:].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def held(cache, row, n):
    """(tokens 0 .. n - 1 of a table row [n, hkv, 128] float64, there [n])."""
    page = cache.shape[1]
    p = torch.arange(max(n, 0))
    bi = p // page
    blk = row[bi.clamp(max=len(row) - 1)].long() if len(row) else torch.full_like(p, -1)
    there = (bi < len(row)) & (blk >= 0) & (blk < cache.shape[0])
    return cache[blk.clamp(0, cache.shape[0] - 1), p % page].double(), there


def store(cache, bt, lens, cu, x):
    """x [tokens, hkv, 128] as own tokens lens[s] .. of every sequence."""
    page = cache.shape[1]
    for s in range(len(cu) - 1):
        for i in range(int(cu[s + 1] - cu[s])):
            p = int(lens[s]) + i
            if p < 0 or p // page >= bt.shape[1]:
                continue
            b = int(bt[s, p // page])
            if 0 <= b < cache.shape[0]:
                cache[b, p % page] = x[int(cu[s]) + i]


def attend(q, kc, vc, pt, plens, cg, bt, lens, cu, scale):
    """(out, weight) [tokens, hq, 128] float64 of rotated q; weight = sum of p
    |v|, what errors of the probabilities are relative to."""
    T, hq, _ = q.shape
    G = hq // kc.shape[2]
    out = torch.zeros(T, hq, 128, dtype=torch.float64)
    wt = torch.zeros_like(out)
    for s in range(len(cu) - 1):
        t0, n = int(cu[s]), int(cu[s + 1] - cu[s])
        c = int(lens[s])
        g = [i for i in range(len(plens)) if cg[i] <= s < cg[i + 1]]
        P = min(max(int(plens[g[0]]), 0), pt.shape[1] * kc.shape[1]) if g else 0
        (pk, pth), (pv, _) = (held(x, pt[g[0]], P) if g else held(x, bt[0][:0], 0) for x in (kc, vc))
        (ok, oth), (ov, _) = (held(x, bt[s], c + n) for x in (kc, vc))
        k, v, there = torch.cat([pk, ok]), torch.cat([pv, ov]), torch.cat([pth, oth])
        for i in range(n):
            see = there & (torch.arange(len(there)) < P + max(c + i + 1, 0))
            if not see.any():
                continue
            ks, vs = k[see], v[see]
            for h in range(hq):
                p = torch.softmax((ks[:, h // G] @ q[t0 + i, h].double()) * scale, 0)
                out[t0 + i, h] = p @ vs[:, h // G]
                wt[t0 + i, h] = p @ vs[:, h // G].abs()
    return out, wt
