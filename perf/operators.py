"""Measured cases of the 4-bit KV cache and of the verification of drafted tokens.

append   new tokens' keys (rotated to their positions) and values into a paged
         cache held in 4 bits, the queries rotated beside them; the appended
         tokens are read back as the values they are held as
read     a stretch of cached tokens as bf16
attend   causal grouped-head attention of new tokens over that cache: single
         tokens, drafted tokens, whole prompts and mixed batches
verify   drafted tokens accepted against the target's probabilities, and the
         next token drawn, from given random numbers

Heads have 128 dims.  The cache is uint8 [blocks, kv heads, page / 16, 2176]: a
record holds 16 tokens of one head.  A group of 32 dims of a token's key or
value is 32 codes (sign, then 0 .5 1 1.5 2 3 4 6) times 2^(b - 127) of one
byte b; b = 255 marks a group with an infinity or a NaN.
  bytes 0..1023     key codes: token t, dim d at 64 t + d / 2, even dims low
  bytes 1024..2047  value codes: 256 (t / 4) + 16 (d / 8) + 4 (t % 4) + d % 8 / 2
  bytes 2048..2111  key scales: 16 (d / 32) + t
  bytes 2112..2175  value scales: 16 (t / 4) + 4 (d / 32) + t % 4
"""

import math
import random

import numpy as np
import torch

own = False

D = 128
TILE = 16        # tokens of a record
REC = 2176       # bytes of a record
THETA = 500000.0
DEV = "cuda"
MAGS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step's tokens of 28 requests, queries rotated beside them
        {"name": "append_28x1", "op": "append", "heads": 32, "kv_heads": 8, "page": 16, "seqs": 28, "new_min": 1,
         "new_max": 1, "ctx_min": 128, "ctx_max": 2048, "shape": 1},
        # packed prompts of different lengths, some behind cached tokens
        {"name": "append_prompts", "op": "append", "heads": 32, "kv_heads": 8, "page": 32, "seqs": 6, "new_min": 1,
         "new_max": 4096, "ctx_min": 1, "ctx_max": 1000, "shape": 2},
        # one short request handed on in bf16
        {"name": "read_short", "op": "read", "kv_heads": 8, "page": 16, "seqs": 1, "new_min": 300, "new_max": 300,
         "ctx_min": 1, "ctx_max": 40, "shape": 3},
        # a few long ones
        {"name": "read_long", "op": "read", "kv_heads": 8, "page": 64, "seqs": 4, "new_min": 9000, "new_max": 32768,
         "ctx_min": 1, "ctx_max": 40, "shape": 4},
        # four requests just begun: latency
        {"name": "attend_token_4", "op": "attend", "heads": 32, "kv_heads": 8, "page": 16, "seqs": 4, "new_min": 1,
         "new_max": 1, "ctx_min": 1, "ctx_max": 300, "many": 0, "shape": 5},
        # the ordinary decode step: 28 requests of 128 to 2048 tokens
        {"name": "attend_token_28", "op": "attend", "heads": 32, "kv_heads": 8, "page": 16, "seqs": 28, "new_min": 1,
         "new_max": 1, "ctx_min": 128, "ctx_max": 2048, "many": 0, "shape": 6},
        # long contexts
        {"name": "attend_token_long", "op": "attend", "heads": 32, "kv_heads": 8, "page": 64, "seqs": 32,
         "new_min": 1, "new_max": 1, "ctx_min": 8192, "ctx_max": 32767, "many": 0, "shape": 7},
        # drafted tokens, another number of them in every request
        {"name": "attend_drafts_28", "op": "attend", "heads": 32, "kv_heads": 8, "page": 16, "seqs": 28,
         "new_min": 1, "new_max": 6, "ctx_min": 128, "ctx_max": 8192, "many": 0, "shape": 8},
        # whole prompts from one token to 8192, nothing cached before them
        {"name": "attend_prompts", "op": "attend", "heads": 32, "kv_heads": 8, "page": 16, "seqs": 5, "new_min": 1,
         "new_max": 8192, "ctx_min": 0, "ctx_max": 0, "many": 0, "shape": 9},
        # a mixed batch: decode tokens beside two prompt chunks of 512
        {"name": "attend_mixed", "op": "attend", "heads": 32, "kv_heads": 8, "page": 32, "seqs": 26, "new_min": 1,
         "new_max": 1, "ctx_min": 200, "ctx_max": 12000, "many": 2, "shape": 10},
        # one request, four tokens drafted by looking them up (no draft distribution)
        {"name": "verify_lookup_1", "op": "verify", "vocab": 32000, "seqs": 1, "new_min": 4, "new_max": 4,
         "drafter": False, "greedy": 0.0, "shape": 11},
        # 28 requests with one to five drafted tokens each, a quarter of them greedy
        {"name": "verify_28", "op": "verify", "vocab": 128256, "seqs": 28, "new_min": 1, "new_max": 5,
         "drafter": True, "greedy": 0.25, "shape": 12},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "attend", "attend", "verify", "verify"])
    shape = rng.randrange(1 << 30)
    while True:
        if op == "verify":
            case = {"op": op, "vocab": rng.choice([_log_int(rng, 1000, 128256), 32000, 128256]),
                    "seqs": _log_int(rng, 1, 64), "new_min": rng.randrange(0, 3), "new_max": rng.randrange(3, 9),
                    "drafter": rng.random() < 0.7, "greedy": rng.choice([0.0, 0.0, 0.25, 1.0]), "shape": shape}
        else:
            kv = rng.choice([1, 2, 4, 8])
            case = {"op": op, "kv_heads": kv, "page": rng.choice([16, 32, 48, 64]), "shape": shape}
            if op != "read":
                case["heads"] = kv * rng.choice([1, 2, 3, 4, 4, 7, 8])
            if op == "read":
                new = _log_int(rng, 1, 32768)
                case.update(seqs=_log_int(rng, 1, 16), new_min=max(1, new // 4), new_max=new, ctx_min=0, ctx_max=100)
            elif op == "append":
                new = _log_int(rng, 1, 4096)
                case.update(seqs=_log_int(rng, 1, 64), new_min=max(1, new // 8), new_max=new, ctx_min=0,
                            ctx_max=_log_int(rng, 1, 4096))
            else:
                kind = rng.choice(["token", "token", "drafts", "prompts", "mixed"])
                ctx = _log_int(rng, 1, 32767)
                seqs = _log_int(rng, 1, 64)
                case.update(many=0, new_min=1, new_max=1, ctx_min=ctx // 8, ctx_max=ctx)
                if kind == "drafts":
                    case["new_max"] = rng.randrange(2, 9)
                elif kind == "prompts":
                    seqs = _log_int(rng, 1, 8)
                    case["new_max"] = _log_int(rng, 16, 8192)
                    if rng.random() < 0.5:
                        case.update(ctx_min=0, ctx_max=0)
                elif kind == "mixed":
                    case["many"] = rng.randrange(1, 4)
                case["seqs"] = seqs
        if _cost(case) <= max(_cost(c) for c in listed() if c["op"] == op):
            return case


def _cost(case):
    """Seconds of a pass at about this card's rates."""
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 1e15)


def _lens(case):
    """New tokens and cached tokens of every sequence, from the case alone."""
    rng = random.Random(case["shape"])
    new = [_log_int(rng, max(case["new_min"], 1), case["new_max"]) if case["new_max"] > 8 else
           rng.randint(case["new_min"], case["new_max"]) for _ in range(case["seqs"])]
    if case["new_max"] > 8:  # the longest of the range is always met
        new[rng.randrange(len(new))] = case["new_max"]
    for i in range(case.get("many", 0)):
        new[(7 * i + 1) % len(new)] = 512
    ctx = [rng.randint(case["ctx_min"], case["ctx_max"]) for _ in new] if "ctx_max" in case else None
    return new, ctx


# ------------------------------------------------------------------ prepare
def _tables(lens, page, gen):
    """Pages of every sequence: a permutation of the pool, unused entries 0."""
    need = [(n + page - 1) // page for n in lens]
    perm = torch.randperm(sum(need) + 1, generator=gen, device=DEV).to(torch.int32)
    bt = torch.zeros(len(lens), max(need), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        bt[i, :n] = perm[at:at + n]
        at += n
    return bt, sum(need) + 1


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _channels(gen, heads):
    """Keys have some channels much larger than others."""
    return torch.exp(0.5 * _randn(gen, heads, D))


def _i32(vals):
    return torch.tensor(vals, dtype=torch.int32, device=DEV)


def _prefix(counts):
    return _i32(np.concatenate([[0], np.cumsum(counts)]).tolist())


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    new, ctx = _lens(case)
    st = {"op": case["op"], "new": new, "ctx": ctx}
    if case["op"] == "verify":
        return _prepare_verify(case, st, gen)
    hkv = case["kv_heads"]
    total = [c + n for c, n in zip(ctx, new)]
    bt, nb = _tables(total, case["page"], gen)
    pages = torch.zeros(nb, hkv, case["page"] // TILE, REC, dtype=torch.uint8, device=DEV)
    chan = _channels(gen, hkv)
    T = sum(new)
    st.update(pages=pages, bt=bt, lens=_i32(ctx), cu=_prefix(new), T=T, max_new=max(new), scale=1.0 / math.sqrt(D))
    fill = total if case["op"] != "append" else ctx
    for s, n in enumerate(fill):
        for a in range(0, n, 8192):
            m = min(n, a + 8192) - a
            k, v = _randn(gen, m, hkv, D) * chan, _randn(gen, m, hkv, D)
            at = torch.arange(a, a + m, device=DEV)
            _store(pages, bt[s, at // case["page"]], at, _quantise(k), _quantise(v))
    if case["op"] == "read":
        return st
    hq = case["heads"]
    if case["op"] == "attend":
        st["q"] = (1.5 * _randn(gen, T, hq, D)).to(torch.bfloat16)
        return st
    qkv = _randn(gen, T, (hq + 2 * hkv) * D)  # the fused projection's rows, heads read in place
    qkv[:, hq * D:(hq + hkv) * D] *= chan.reshape(-1)
    st["qkv"] = qkv = qkv.to(torch.bfloat16)
    st["q"] = qkv[:, :hq * D].view(T, hq, D)
    st["k"] = qkv[:, hq * D:(hq + hkv) * D].view(T, hkv, D)
    st["v"] = qkv[:, (hq + hkv) * D:].view(T, hkv, D)
    st["pos"] = torch.cat([torch.arange(c, c + n, device=DEV) for c, n in zip(ctx, new)])
    ang = torch.outer(torch.arange(max(total), device=DEV, dtype=torch.float64),
                      THETA ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D))
    st["cos_sin"] = torch.cat([ang.cos(), ang.sin()], -1).to(torch.bfloat16).contiguous()
    return st


def _prepare_verify(case, st, gen):
    """Target logits with a few likely tokens in every row; the drafter's are
    near them, and the drafted tokens are drawn from the drafter's (or are the
    target's likely ones, now and then another, without a drafter)."""
    new, V, n = st["new"], case["vocab"], case["seqs"]
    rows, T = sum(new) + n, sum(new)
    logits = 2.0 * _randn(gen, rows, V)
    for _ in range(6):
        at = torch.randint(V, (rows, 1), generator=gen, device=DEV)
        logits.scatter_add_(1, at, 4.0 + 8.0 * torch.rand(rows, 1, generator=gen, device=DEV))
    temp = 0.6 + 0.6 * torch.rand(n, generator=gen, device=DEV)
    temp[torch.rand(n, generator=gen, device=DEV) < case["greedy"]] = 0.0
    row = [sum(new[:s]) + s + j for s in range(n) for j in range(new[s])]
    drow = torch.tensor(row, dtype=torch.int64, device=DEV)
    seq = torch.tensor([s for s in range(n) for _ in range(new[s])], dtype=torch.int64, device=DEV)
    st.update(logits=logits.to(torch.bfloat16), temp=temp, cu=_prefix(new), T=T, max_new=max(new), drafts=None,
              u=torch.rand(T, generator=gen, device=DEV), u_last=torch.rand(n, generator=gen, device=DEV))
    near = logits[drow] + 0.7 * _randn(gen, T, V)
    t = temp[seq].clamp(min=1e-3).unsqueeze(1)
    noise = -torch.log(-torch.log(torch.rand(T, V, generator=gen, device=DEV).clamp(1e-20, 1 - 1e-7)))
    if case["drafter"]:
        st["drafts"] = near.to(torch.bfloat16)
        near = st["drafts"].float()
    st["ids"] = (near / t + noise).argmax(-1) if T else torch.zeros(0, dtype=torch.int64, device=DEV)
    return st


# ------------------------------------------------------------ the plain form
def _quantise(x):
    """Codes (uint8, a dim each) and scale bytes of x [..., 128] fp32."""
    g = x.reshape(*x.shape[:-1], D // 32, 32)
    top = g.abs().amax(-1)
    b = (((top.view(torch.int32) + 0x200000) >> 23) - 2).clamp(2, 252)
    b = torch.where(torch.isfinite(top), b, torch.full_like(b, 255))
    unit = ((254 - b.clamp(max=252)) << 23).view(torch.float32).unsqueeze(-1)
    m = (g * unit).abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
    code = code + 8 * torch.signbit(g).to(torch.uint8)
    return code.reshape(x.shape), b.to(torch.uint8)


def _values(code, b):
    """The fp32 values of codes [..., 128] under scale bytes [..., 4]."""
    lut = torch.tensor(MAGS + tuple(-m for m in MAGS), device=code.device)
    scale = torch.where(b == 255, torch.full_like(b, 1, dtype=torch.float32) * math.nan,
                        (b.to(torch.int32) << 23).view(torch.float32))
    return (lut[code.int()].reshape(*code.shape[:-1], D // 32, 32) * scale.unsqueeze(-1)).reshape(code.shape)


def _store(pages, block, at, k, v):
    """Tokens at positions `at` of their sequences, in pages `block`; k / v =
    codes and scales of [tokens, kv heads, 128]."""
    hkv, page = pages.shape[1], pages.shape[2] * TILE
    rec = (block.long() * hkv).unsqueeze(1) + torch.arange(hkv, device=at.device)  # [tokens, heads]
    base = ((rec * (page // TILE) + (at % page // TILE).unsqueeze(1)) * REC).unsqueeze(-1)
    t = (at % TILE).view(-1, 1, 1)
    flat = pages.view(-1)
    byte = torch.arange(64, device=at.device)
    grp = torch.arange(4, device=at.device)
    pack = lambda c: c[..., 0::2] | (c[..., 1::2] << 4)  # noqa: E731
    flat[base + 64 * t + byte] = pack(k[0])
    flat[base + 1024 + 256 * (t // 4) + 16 * (byte // 4) + 4 * (t % 4) + byte % 4] = pack(v[0])
    flat[base + 2048 + 16 * grp + t] = k[1]
    flat[base + 2112 + 16 * (t // 4) + 4 * grp + t % 4] = v[1]


def _load(pages, table, n):
    """Keys and values [kv heads, n, 128] fp32 of a sequence's first n tokens."""
    hkv, page = pages.shape[1], pages.shape[2] * TILE
    r = pages[table[:(n + page - 1) // page].long()].transpose(0, 1).reshape(hkv, -1, REC)[:, :(n + TILE - 1) // TILE]
    nt = r.shape[1]
    split = lambda c: torch.stack([c & 15, c >> 4], -1).reshape(hkv, nt * TILE, D)[:, :n]  # noqa: E731
    kc = split(r[..., :1024].reshape(hkv, nt * TILE, 64))
    vc = split(r[..., 1024:2048].reshape(hkv, nt, 4, 16, 4, 4).permute(0, 1, 2, 4, 3, 5).reshape(hkv, nt * TILE, 64))
    ks = r[..., 2048:2112].reshape(hkv, nt, 4, TILE).transpose(2, 3).reshape(hkv, nt * TILE, 4)[:, :n]
    vs = r[..., 2112:].reshape(hkv, nt, 4, 4, 4).transpose(3, 4).reshape(hkv, nt * TILE, 4)[:, :n]
    return _values(kc, ks), _values(vc, vs)


def _rotate(x, cs):
    """Halves (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin), fp32."""
    a, b = x[..., :D // 2].float(), x[..., D // 2:].float()
    c, s = cs[:, None, :D // 2], cs[:, None, D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _plain_read(st):
    out = [_load(st["pages"], st["bt"][s], c + n) for s, (c, n) in enumerate(zip(st["ctx"], st["new"]))]
    return [torch.cat([o[i][:, c:].transpose(0, 1) for o, c in zip(out, st["ctx"])]).to(torch.bfloat16)
            for i in (0, 1)]


def _sequences(st):
    """The sequence of every packed token."""
    return torch.searchsorted(st["cu"][1:].long(), torch.arange(st["T"], device=DEV), right=True)


def _plain_append(st):
    cs = st["cos_sin"][st["pos"]].float()
    q = _rotate(st["q"], cs).to(torch.bfloat16)
    k, v = _quantise(_rotate(st["k"], cs)), _quantise(st["v"].float())
    seq = _sequences(st)
    at = st["lens"].long()[seq] + torch.arange(st["T"], device=DEV) - st["cu"].long()[seq]
    _store(st["pages"], st["bt"][seq, at // (st["pages"].shape[2] * TILE)], at, k, v)
    return [q, _values(*k).to(torch.bfloat16), _values(*v).to(torch.bfloat16)]


def _plain_attend(st):
    q = st["q"]
    hq = q.shape[1]
    out = torch.empty(q.shape[0], hq * D, dtype=torch.bfloat16, device=DEV)
    at = 0
    for s, (c, n) in enumerate(zip(st["ctx"], st["new"])):
        k, v = _load(st["pages"], st["bt"][s], c + n)
        hkv = k.shape[0]
        for a in range(0, n, 1024):
            m = min(n, a + 1024) - a
            see = c + a + m
            x = q[at + a:at + a + m].float().view(m, hkv, hq // hkv, D).transpose(0, 1).reshape(hkv, -1, D)
            w = torch.matmul(x, k[:, :see].transpose(1, 2)).view(hkv, m, hq // hkv, see) * st["scale"]
            if m > 1:
                hide = torch.arange(see, device=DEV) > torch.arange(c + a, see, device=DEV).unsqueeze(1)
                w = w.masked_fill(hide[None, :, None, :], -math.inf)
            w = torch.exp(w - w.amax(-1, keepdim=True))
            w = w / w.sum(-1, keepdim=True)
            o = torch.matmul(w.view(hkv, -1, see), v[:, :see])
            out[at + a:at + a + m] = o.view(hkv, m, -1, D).transpose(0, 1).reshape(m, hq * D).to(torch.bfloat16)
        at += n
    return out


def _plain_verify(st):
    dev = DEV
    n, T, V = st["temp"].shape[0], st["T"], st["logits"].shape[1]
    seq = _sequences(st)
    step = torch.arange(T, device=dev) - st["cu"][:-1].long()[seq]
    first = st["cu"][:-1].long() + torch.arange(n, device=dev)  # a sequence's first target row
    temp = st["temp"].double()
    greedy = temp <= 0

    def probs(rows, of):
        x = rows.double() / torch.where(greedy, 1.0, temp)[of].unsqueeze(1)
        e = torch.exp(x - x.amax(-1, keepdim=True))
        return e / e.sum(-1, keepdim=True)

    ids, drow = st["ids"], first[seq] + step
    tgt = st["logits"][drow]
    p = probs(tgt, seq)
    pd = p.gather(1, ids.unsqueeze(1)).squeeze(1)
    q = probs(st["drafts"], seq) if st["drafts"] is not None else None
    qd = q.gather(1, ids.unsqueeze(1)).squeeze(1) if q is not None else torch.ones_like(pd)
    ok = torch.where(greedy[seq], tgt.float().argmax(-1) == ids, st["u"].double() * qd < pd)
    acc = torch.zeros(n, st["max_new"] + 1, dtype=torch.int64, device=dev)
    acc[seq, step] = ok.long()
    acc = acc.cumprod(1).sum(1)  # drafts before the first refused one
    count = (st["cu"][1:] - st["cu"][:-1]).long()
    last = st["logits"][first + acc]
    w = probs(last, torch.arange(n, device=dev))
    if T:
        refused = (acc < count) & ~greedy
        j = (st["cu"][:-1].long() + acc).clamp(max=T - 1)
        if q is not None:
            less = q[j]
        else:
            less = torch.zeros_like(w).scatter_(1, ids[j].unsqueeze(1), math.inf)
        w = torch.where(refused.unsqueeze(1), (w - less).clamp(min=0.0), w)
    c = w.cumsum(-1)
    pick = (c <= st["u_last"].double().unsqueeze(1) * c[:, -1:]).sum(-1).clamp(max=V - 1)
    pick = torch.where(greedy, last.float().argmax(-1), pick)
    out = torch.full((n, st["max_new"] + 1), -1, dtype=torch.int64, device=dev)
    out[seq, step] = torch.where(step < acc[seq], ids, -1)
    out[torch.arange(n, device=dev), acc] = pick
    return [out, acc.to(torch.int32)]


# ---------------------------------------------------------------------- run
def run(st):
    op = st["op"]
    if own:
        from swarmlora_amd import ops
        if op == "append":
            q = ops.kv4_append(st["k"], st["v"], st["pages"], st["bt"], st["lens"], st["pos"], st["cos_sin"],
                               q=st["q"], cu_seqlens=st["cu"])
            k, v = ops.kv4_read(st["pages"], st["bt"], st["lens"], st["T"], cu_seqlens=st["cu"])
            return [q, k, v]
        if op == "read":
            return list(ops.kv4_read(st["pages"], st["bt"], st["lens"], st["T"], cu_seqlens=st["cu"]))
        if op == "attend":
            return ops.kv4_attention(st["q"], st["pages"], st["bt"], st["lens"], st["scale"], cu_seqlens=st["cu"],
                                     max_q_len=st["max_new"])
        return list(ops.verify_drafts(st["logits"], st["ids"], st["u"], st["u_last"], st["temp"],
                                      draft_logits=st["drafts"], cu_drafts=st["cu"], max_drafts=st["max_new"]))
    return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend, "verify": _plain_verify}[op](st)


def work(case):
    new, ctx = _lens(case)
    T = sum(new)
    if case["op"] == "verify":
        rows = T + len(new) + (T if case["drafter"] else 0)
        return {"bytes": rows * case["vocab"] * 2 + T * 20 + len(new) * 20, "flops": rows * case["vocab"] * 4}
    held = case["kv_heads"] * 2 * (D // 2 + D // 32)  # bytes of a token in the cache
    if case["op"] == "read":
        return {"bytes": T * (held + case["kv_heads"] * 4 * D), "flops": T * case["kv_heads"] * 2 * D}
    if case["op"] == "append":
        hq, hkv = case["heads"], case["kv_heads"]
        # rows in, rotated queries out, the cache written and read back, the values out
        return {"bytes": T * ((hq + 2 * hkv) * 2 * D + hq * 2 * D + 2 * held + hkv * 4 * D + 2 * D + 8),
                "flops": T * (hq + 2 * hkv) * 3 * D}
    hq = case["heads"]
    seen = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, ctx))
    return {"bytes": sum(c + n for c, n in zip(ctx, new)) * held + T * hq * 4 * D, "flops": seen * hq * 4 * D}


# -------------------------------------------------------------------- exact
def _held64(pages, table, a, b):
    """Keys and values [tokens a..b, kv heads, 128] in 64 bits, byte by byte
    of the record's definition."""
    page = pages.shape[2] * TILE
    at = torch.arange(a, b, device=pages.device)
    rec = pages[table[at // page].long(), :, at % page // TILE].long()  # [tokens, heads, bytes]
    t = (at % TILE).view(-1, 1, 1)
    d = torch.arange(D, device=pages.device)
    pick = lambda i: rec.gather(2, i.expand(rec.shape[0], rec.shape[1], D))  # noqa: E731
    mags = torch.tensor(MAGS, dtype=torch.float64, device=pages.device)
    out = []
    for code, scale in ((64 * t + d // 2, 2048 + 16 * (d // 32) + t),
                        (1024 + 256 * (t // 4) + 16 * (d // 8) + 4 * (t % 4) + d % 8 // 2,
                         2112 + 16 * (t // 4) + 4 * (d // 32) + t % 4)):
        c = (pick(code) >> (4 * (d % 2))) % 16
        b8 = pick(scale).double()
        x = mags[c % 8] * torch.where(c >= 8, -1.0, 1.0) * torch.exp2(b8 - 127)
        out.append(torch.where(b8 == 255, math.nan, x))
    return out


def _nearest64(x):
    """x [.., 128] in 64 bits, each group of 32 on its grid."""
    g = x.unflatten(-1, (D // 32, 32))
    top = g.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=1e-300)))
    e = e + (top >= 1.75 * torch.exp2(e)).double() - 2
    e = e.clamp(2 - 127, 252 - 127)
    y = (g.abs() / torch.exp2(e)).clamp(max=6.0)
    # spacing 0.5 up to 2, 1 up to 4, 2 up to 6; round half to even
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    return (torch.copysign(torch.round(y / step) * step, g) * torch.exp2(e)).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    new, ctx = st["new"], st["ctx"]
    if case["op"] == "verify":
        return _exact_verify(st)
    if case["op"] == "append":
        cs = st["cos_sin"][st["pos"]].double()
        turn = torch.complex(cs[:, :D // 2], cs[:, D // 2:]).unsqueeze(1)

        def rot(x):
            z = torch.complex(x[..., :D // 2].double(), x[..., D // 2:].double()) * turn
            return torch.cat([z.real, z.imag], -1)
        return [rot(st["q"]), _nearest64(rot(st["k"])), _nearest64(st["v"].double())]
    if case["op"] == "read":
        got = [[], []]
        for s, (c, n) in enumerate(zip(ctx, new)):
            for a in range(c, c + n, 2048):
                for lst, x in zip(got, _held64(st["pages"], st["bt"][s], a, min(c + n, a + 2048))):
                    lst.append(x)
        return [torch.cat(g) for g in got]
    q, hq = st["q"].double(), st["q"].shape[1]
    hkv = st["pages"].shape[1]
    rows = []
    at = 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        kv = [_held64(st["pages"], st["bt"][s], a, min(c + n, a + 2048)) for a in range(0, c + n, 2048)]
        k, v = (torch.cat([x[i] for x in kv]) for i in (0, 1))
        res = torch.empty(n, hq, D, dtype=torch.float64, device=DEV)
        for h in range(hq):
            kh, vh = k[:, h * hkv // hq], v[:, h * hkv // hq]
            for a in range(0, n, 2048):
                i = torch.arange(a, min(n, a + 2048), device=DEV)
                sc = (q[at + i, h] @ kh.T) * st["scale"]
                sc[torch.arange(c + n, device=DEV) > (c + i).unsqueeze(1)] = -math.inf
                res[i, h] = torch.softmax(sc, -1) @ vh
        rows.append(res.flatten(1))
        at += n
    return torch.cat(rows)


def _exact_verify(st):
    """One sequence after another, as the rule reads."""
    toks, counts = [], []
    at = row = 0
    for s, n in enumerate(st["new"]):
        t = float(st["temp"][s])
        take, out = n, [-1] * (st["max_new"] + 1)
        less = None
        for j in range(n):
            x, d = st["logits"][row + j].double(), int(st["ids"][at + j])
            if t <= 0:
                ok = int(x.float().argmax()) == d
            else:
                p = torch.softmax(x / t, 0)
                q = torch.softmax(st["drafts"][at + j].double() / t, 0) if st["drafts"] is not None else None
                ok = float(st["u"][at + j]) * (float(q[d]) if q is not None else 1.0) < float(p[d])
            if not ok:
                take = j
                if t > 0:
                    less = q if q is not None else torch.zeros_like(p).index_fill_(0, torch.tensor([d], device=DEV), 2.0)
                break
            out[j] = d
        x = st["logits"][row + take].double()
        if t <= 0:
            out[take] = int(x.float().argmax())
        else:
            w = torch.softmax(x / t, 0)
            if less is not None:
                w = (w - less).clamp(min=0)
            c = np.cumsum(w.cpu().numpy())
            out[take] = int(np.searchsorted(c, float(st["u_last"][s]) * c[-1], side="right"))
        toks.append(out)
        counts.append(take)
        at += n
        row += n + 1
    return [torch.tensor(toks), torch.tensor(counts, dtype=torch.int32)]
