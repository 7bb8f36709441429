"""The 4-bit KV cache from its definition, in 64 bits on the CPU: encoding and
decoding of records, append, and attention."""

import math

import torch

MAGS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
REC = 2176


def encode(x):
    """x [..., 128] float64 -> (codes [..., 128], scale bytes [..., 4])."""
    g = x.unflatten(-1, (4, 32))
    top = g.abs().amax(-1)
    ok = torch.isfinite(g).all(-1)
    b = torch.full(top.shape, 2, dtype=torch.int64)
    for e in range(3, 253):  # the least b with the largest under 7 * 2^(b - 127)
        b = torch.where(top >= 7 * 2.0 ** (e - 1 - 127), e, b)
    y = (g.abs() / torch.exp2(b.double() - 127).unsqueeze(-1)).nan_to_num(0.0, 6.0)
    d = (y.clamp(max=6.0).unsqueeze(-1) - MAGS).abs()
    near = d.amin(-1, keepdim=True)
    even = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])  # ties to the even code: it comes first
    code = even[(d[..., even] == near).int().argmax(-1)]
    code = code + 8 * torch.signbit(g).long()
    return code.flatten(-2), torch.where(ok, b, 255)


def decode(code, b):
    x = MAGS[code % 8] * torch.where(code >= 8, -1.0, 1.0).double()
    s = torch.where(b == 255, math.nan, torch.exp2(b.double() - 127))
    return (x.unflatten(-1, (4, 32)) * s.unsqueeze(-1)).flatten(-2)


def code_at(t, d, value):
    """Byte and shift of token t's (0..15) dim d in a record."""
    if value:
        return 1024 + 256 * (t // 4) + 16 * (d // 8) + 4 * (t % 4) + d % 8 // 2, 4 * (d % 2)
    return 64 * t + d // 2, 4 * (d % 2)


def scale_at(t, g, value):
    return 2112 + 16 * (t // 4) + 4 * g + t % 4 if value else 2048 + 16 * g + t


_D = torch.arange(128)


def place(bt, page, num_blocks, s, p):
    """(block, record of the page, token of the record) of token p, or None."""
    if p < 0 or p // page >= bt.shape[1]:
        return None
    b = int(bt[s, p // page])
    return (b, p % page // 16, p % 16) if 0 <= b < num_blocks else None


def store(pages, bt, s, p, k, v):
    """k, v [hkv, 128] float64 as token p of sequence s."""
    at = place(bt, pages.shape[2] * 16, pages.shape[0], s, p)
    if at is None:
        return
    b, r, t = at
    for value, x in ((False, k), (True, v)):
        code, sc = encode(x)
        byte, sh = code_at(t, _D, value)
        rec = pages[b, :, r]
        rec[:, byte[::2]] = (code[:, ::2] | code[:, 1::2] << 4).to(torch.uint8)
        rec[:, scale_at(t, torch.arange(4), value)] = sc.to(torch.uint8)


def load(pages, bt, s, n):
    """(k, v [n, hkv, 128] float64, there [n])."""
    hkv = pages.shape[1]
    page = pages.shape[2] * 16
    p = torch.arange(n)
    bi = p // page
    blk = bt[s][bi.clamp(max=bt.shape[1] - 1)].long()
    there = (bi < bt.shape[1]) & (blk >= 0) & (blk < pages.shape[0])
    rec = pages[blk.clamp(0, pages.shape[0] - 1), :, p % page // 16].long()  # [n, hkv, REC]
    t = (p % 16).view(-1, 1)
    out = []
    for value in (False, True):
        byte, sh = code_at(t, _D, value)
        code = rec.gather(2, byte.unsqueeze(1).expand(n, hkv, 128)) >> sh.unsqueeze(0 if sh.dim() < 2 else 1) & 15
        b = rec.gather(2, scale_at(t, torch.arange(4), value).unsqueeze(1).expand(n, hkv, 4))
        out.append(decode(code, b))
    return out[0], out[1], there


def rotate(x, cs):
    """NeoX halves of x [..., heads, 128] at cs [..., 128] = cos | sin."""
    a, b = x[..., :64].double(), x[..., 64:].double()
    c, s = cs[..., None, :64].double(), cs[..., None, 64:].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def attend(q, pages, bt, lens, cu, scale, used=None):
    """(out, weight) [tokens, hq, 128] float64; weight = sum of p |v|, what
    errors of the probabilities are relative to."""
    T, hq, _ = q.shape
    hkv = pages.shape[1]
    G = hq // hkv
    out = torch.zeros(T, hq, 128, dtype=torch.float64)
    wt = torch.zeros_like(out)
    for s in range(len(cu) - 1):
        n = int(cu[s + 1] - cu[s])
        if n == 0:
            continue
        c = int(lens[s])
        if c + n <= 0:
            continue
        k, v, there = load(pages, bt, s, c + n)
        i = torch.arange(n)
        see = (torch.arange(c + n) <= c + i.unsqueeze(1)) & there  # [n, keys]
        v = torch.where(there.view(-1, 1, 1), v, 0.0)
        for h in range(hkv):
            x = q[cu[s]:cu[s] + n, h * G:(h + 1) * G].double()  # [n, G, 128]
            sc = (x @ k[:, h].T) * scale
            sc = torch.where(see.unsqueeze(1), sc, -math.inf)
            m = sc.amax(-1, keepdim=True)
            p = torch.exp(sc - torch.where(m == -math.inf, 0.0, m))
            p = p / p.sum(-1, keepdim=True)
            p = torch.where(see.any(-1).view(n, 1, 1), p, 0.0)
            # a NaN value reaches the queries that see it, nobody else
            bad = torch.isnan(v[:, h])
            nan = (see.double() @ bad.double() > 0).unsqueeze(1)
            vz = torch.where(bad, 0.0, v[:, h])
            o = p @ vz
            out[cu[s]:cu[s] + n, h * G:(h + 1) * G] = torch.where(nan, math.nan, o)
            wt[cu[s]:cu[s] + n, h * G:(h + 1) * G] = p @ vz.abs()
    return out, wt
