"""Measured cases of attention over a shared prefix, of sampling from given
random numbers and of products in 8-bit integers.

share    causal grouped-head attention of new tokens of several sequences over
         a prefix that a group of sequences shares and the pages of their own;
         the new keys are rotated to their positions and stored with the values
sample   the next token of every row of logits: temperature, top-k, top-p and
         min-p, drawn from given random numbers
int8     rows made 8-bit integers with a scale each, times a weight held in
         8-bit integers with a scale for each output channel

Heads have 128 dims; the caches are bf16 [blocks, page, kv heads, 128].
"""

import math
import random

import numpy as np
import torch

own = False

D = 128
THETA = 500000.0
DEV = "cuda"
BF16 = torch.bfloat16


# ------------------------------------------------------------------- cases
def listed():
    return [
        # four answers to one question, just begun: latency
        {"name": "share_token_4", "op": "share", "heads": 32, "kv_heads": 8, "page": 16, "groups": 1, "seqs": 4,
         "new_min": 1, "new_max": 1, "pre_min": 700, "pre_max": 700, "ctx_min": 0, "ctx_max": 20, "shape": 1},
        # the ordinary decode step: 32 requests behind one system prompt
        {"name": "share_token_32", "op": "share", "heads": 32, "kv_heads": 8, "page": 16, "groups": 1, "seqs": 32,
         "new_min": 1, "new_max": 1, "pre_min": 4096, "pre_max": 4096, "ctx_min": 1, "ctx_max": 512, "shape": 2},
        # six tenants, each with a prompt of its own before its requests
        {"name": "share_tenants_48", "op": "share", "heads": 32, "kv_heads": 8, "page": 32, "groups": 6, "seqs": 48,
         "new_min": 1, "new_max": 1, "pre_min": 300, "pre_max": 12000, "ctx_min": 16, "ctx_max": 2000, "shape": 3},
        # drafted tokens, another number of them in every request
        {"name": "share_drafts_28", "op": "share", "heads": 32, "kv_heads": 8, "page": 16, "groups": 1, "seqs": 28,
         "new_min": 1, "new_max": 6, "pre_min": 8191, "pre_max": 8191, "ctx_min": 100, "ctx_max": 1000, "shape": 4},
        # questions of 1 to 1024 tokens about one long document
        {"name": "share_prompts_12", "op": "share", "heads": 32, "kv_heads": 8, "page": 64, "groups": 1, "seqs": 12,
         "new_min": 1, "new_max": 1024, "pre_min": 8000, "pre_max": 8000, "ctx_min": 0, "ctx_max": 0, "shape": 5},
        # one request with a small vocabulary, top-p alone
        {"name": "sample_1", "op": "sample", "vocab": 32000, "rows": 1, "kind": "top_p", "greedy": 0.0, "shape": 6},
        # a decode step of 28 requests that ask for different things
        {"name": "sample_28", "op": "sample", "vocab": 128256, "rows": 28, "kind": "mixed", "greedy": 0.25, "shape": 7},
        # many short requests, all filters on
        {"name": "sample_256", "op": "sample", "vocab": 128256, "rows": 256, "kind": "all", "greedy": 0.0, "shape": 8},
        # one token through the fused QKV projection
        {"name": "int8_qkv_1", "op": "int8", "m": 1, "n": 6144, "k": 4096, "bias": False, "shape": 9},
        # a decode step's tokens through Gate+Up
        {"name": "int8_gate_up_28", "op": "int8", "m": 28, "n": 28672, "k": 4096, "bias": False, "shape": 10},
        # a short prompt beside a few tokens through Down
        {"name": "int8_down_107", "op": "int8", "m": 107, "n": 4096, "k": 14336, "bias": True, "shape": 11},
        # prompts of sixteen requests through Gate+Up
        {"name": "int8_prefill_2325", "op": "int8", "m": 2325, "n": 28672, "k": 4096, "bias": False, "shape": 12},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["share", "share", "share", "share", "sample", "sample", "int8", "int8"])
    shape = rng.randrange(1 << 30)
    while True:
        if op == "sample":
            case = {"op": op, "vocab": rng.choice([_log_int(rng, 1000, 128256), 32000, 128256]),
                    "rows": _log_int(rng, 1, 256), "kind": rng.choice(["none", "top_k", "top_p", "min_p", "mixed", "all"]),
                    "greedy": rng.choice([0.0, 0.0, 0.25]), "shape": shape}
        elif op == "int8":
            case = {"op": op, "m": rng.choice([_log_int(rng, 1, 64), _log_int(rng, 1, 2325)]),
                    "n": _log_int(rng, 128, 28672), "k": _log_int(rng, 128, 14336), "bias": rng.random() < 0.5,
                    "shape": shape}
        else:
            kv = rng.choice([1, 2, 4, 8])
            seqs = _log_int(rng, 1, 64)
            pre, ctx = _log_int(rng, 1, 16384), _log_int(rng, 1, 4096)
            case = {"op": op, "heads": kv * rng.choice([1, 2, 3, 4, 4, 7, 8]), "kv_heads": kv,
                    "page": rng.choice([8, 16, 16, 24, 32, 64]), "groups": min(seqs, rng.choice([1, 1, 2, 5])),
                    "seqs": seqs, "new_min": 1, "new_max": 1, "pre_min": max(1, pre // 8), "pre_max": pre,
                    "ctx_min": ctx // 8, "ctx_max": ctx, "shape": shape}
            kind = rng.choice(["token", "token", "drafts", "prompts"])
            if kind == "drafts":
                case["new_max"] = rng.randrange(2, 9)
            elif kind == "prompts":
                case["new_max"] = _log_int(rng, 16, 1024)
        if _cost(case) <= max(_cost(c) for c in listed() if c["op"] == op):
            return case


def _cost(case):
    """Seconds of a pass at about this card's rates."""
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 1e15)


def _lens(case):
    """New and cached tokens of every sequence, the groups' prefixes and the
    number of sequences of each, from the case alone."""
    rng = random.Random(case["shape"])
    n, g = case["seqs"], case["groups"]
    new = [_log_int(rng, case["new_min"], case["new_max"]) if case["new_max"] > 8 else
           rng.randint(case["new_min"], case["new_max"]) for _ in range(n)]
    if case["new_max"] > 8:  # the longest of the range is always met
        new[rng.randrange(n)] = case["new_max"]
    ctx = [rng.randint(case["ctx_min"], case["ctx_max"]) for _ in new]
    pre = [_log_int(rng, case["pre_min"], case["pre_max"]) for _ in range(g)]
    cut = sorted(rng.sample(range(1, n), g - 1)) if g > 1 else []
    size = [b - a for a, b in zip([0] + cut, cut + [n])]
    return new, ctx, pre, size


# ------------------------------------------------------------------ prepare
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _i32(vals):
    return torch.tensor(vals, dtype=torch.int32, device=DEV)


def _prefix(counts):
    return _i32(np.concatenate([[0], np.cumsum(counts)]).tolist())


def _tables(lens, page, perm, at):
    """Pages of every sequence from the permutation, unused entries 0."""
    need = [(n + page - 1) // page for n in lens]
    bt = torch.zeros(len(lens), max(1, max(need)), dtype=torch.int32, device=DEV)
    for i, n in enumerate(need):
        bt[i, :n] = perm[at:at + n]
        at += n
    return bt, at


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return {"share": _prepare_share, "sample": _prepare_sample, "int8": _prepare_int8}[case["op"]](case, gen)


def _prepare_share(case, gen):
    new, ctx, pre, size = _lens(case)
    hq, hkv, page, T = case["heads"], case["kv_heads"], case["page"], sum(new)
    total = [c + n for c, n in zip(ctx, new)]
    blocks = sum((n + page - 1) // page for n in pre + total) + 1
    perm = torch.randperm(blocks, generator=gen, device=DEV).to(torch.int32)
    pt, at = _tables(pre, page, perm, 0)
    bt, _ = _tables(total, page, perm, at)
    chan = torch.exp(0.5 * _randn(gen, hkv, D))  # keys have some channels much larger than others
    kc = torch.empty(blocks, page, hkv, D, dtype=BF16, device=DEV)
    vc = torch.empty_like(kc)
    for a in range(0, blocks, 1024):
        b = min(blocks, a + 1024)
        kc[a:b] = _randn(gen, b - a, page, hkv, D) * chan
        vc[a:b] = _randn(gen, b - a, page, hkv, D)
    qkv = _randn(gen, T, (hq + 2 * hkv) * D)  # the fused projection's rows, heads read in place
    qkv[:, hq * D:(hq + hkv) * D] *= chan.reshape(-1)
    qkv = qkv.to(BF16)
    group = [g for g, n in enumerate(size) for _ in range(n)]
    pos = torch.cat([torch.arange(pre[g] + c, pre[g] + c + n, device=DEV) for g, c, n in zip(group, ctx, new)])
    far = max(pre[g] + t for g, t in zip(group, total))
    ang = torch.outer(torch.arange(far, device=DEV, dtype=torch.float64),
                      THETA ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D))
    return {"op": "share", "new": new, "ctx": ctx, "pre": pre, "group": group, "kc": kc, "vc": vc, "pt": pt, "bt": bt,
            "plen": _i32(pre), "lens": _i32(ctx), "cu": _prefix(new), "cg": _prefix(size), "T": T,
            "q": qkv[:, :hq * D].view(T, hq, D), "k": qkv[:, hq * D:(hq + hkv) * D].view(T, hkv, D),
            "v": qkv[:, (hq + hkv) * D:].view(T, hkv, D), "pos": pos, "scale": 1.0 / math.sqrt(D),
            "cos_sin": torch.cat([ang.cos(), ang.sin()], -1).to(BF16).contiguous()}


def _prepare_sample(case, gen):
    """Logits with a few likely tokens in every row, and what each row asks for."""
    n, V, kind = case["rows"], case["vocab"], case["kind"]
    x = 2.0 * _randn(gen, n, V)
    for _ in range(6):
        at = torch.randint(V, (n, 1), generator=gen, device=DEV)
        x.scatter_add_(1, at, 4.0 + 8.0 * torch.rand(n, 1, generator=gen, device=DEV))
    rng = random.Random(case["shape"])
    want = {"none": [""], "top_k": ["k"], "top_p": ["p"], "min_p": ["m"], "all": ["kpm"],
            "mixed": ["", "k", "p", "m", "kp", "pm"]}[kind]
    has = [rng.choice(want) for _ in range(n)]
    temp = 0.6 + 0.8 * torch.rand(n, generator=gen, device=DEV)
    temp[torch.tensor([rng.random() < case["greedy"] for _ in range(n)], device=DEV)] = 0.0
    f32 = lambda vals: torch.tensor(vals, dtype=torch.float32, device=DEV)  # noqa: E731
    return {"op": "sample", "x": x.to(BF16), "temp": temp, "u": torch.rand(n, generator=gen, device=DEV),
            "top_k": _i32([rng.choice([5, 20, 50, 200, 1000]) if "k" in h else 0 for h in has]),
            "top_p": f32([rng.choice([0.5, 0.8, 0.9, 0.95, 0.99]) if "p" in h else 1.0 for h in has]),
            "min_p": f32([rng.choice([0.02, 0.05, 0.1]) if "m" in h else 0.0 for h in has])}


def _weight(case, gen):
    return (0.02 * _randn(gen, case["n"], case["k"]) * torch.exp(0.3 * _randn(gen, case["n"], 1))).to(BF16)


def _activations(case, gen):
    """Rows with a few channels far above the rest, and the bias."""
    x = _randn(gen, case["m"], case["k"])
    x[:, torch.randint(case["k"], (max(1, case["k"] // 512),), generator=gen, device=DEV)] *= 8.0
    return {"op": "int8", "x": x.to(BF16), "bias": _randn(gen, case["n"]).to(BF16) if case["bias"] else None}


def _prepare_int8(case, gen):
    """The weight as a program holds it, made once."""
    w = _weight(case, gen)
    st = _activations(case, gen)
    if own:
        from swarmlora_amd import ops
        st["w"] = ops.Int8Weight(w)
    else:
        st["w"] = _plain_rows(w)
    return st


# ------------------------------------------------------------ the plain form
def _rotate(x, cs):
    """Halves (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin), fp32."""
    a, b = x[..., :D // 2].float(), x[..., D // 2:].float()
    c, s = cs[:, None, :D // 2], cs[:, None, D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _held(cache, table, n):
    """The first n tokens of a table [kv heads, n, 128] in fp32."""
    page = cache.shape[1]
    return cache[table[:(n + page - 1) // page].long()].flatten(0, 1)[:n].transpose(0, 1).float()


def _plain_share(st):
    kc, vc, page = st["kc"], st["vc"], st["kc"].shape[1]
    cs = st["cos_sin"][st["pos"]].float()
    seq = torch.searchsorted(st["cu"][1:].long(), torch.arange(st["T"], device=DEV), right=True)
    at = st["lens"].long()[seq] + torch.arange(st["T"], device=DEV) - st["cu"].long()[seq]
    block = st["bt"][seq, at // page].long()
    kc[block, at % page] = _rotate(st["k"], cs).to(BF16)
    vc[block, at % page] = st["v"]
    q = _rotate(st["q"], cs).to(BF16).float()
    hq, hkv = q.shape[1], kc.shape[2]
    out = torch.empty(st["T"], hq * D, dtype=BF16, device=DEV)
    shared = [[_held(c, st["pt"][g], n) for c in (kc, vc)] for g, n in enumerate(st["pre"])]
    at = 0
    for s, (c, n, g) in enumerate(zip(st["ctx"], st["new"], st["group"])):
        P = st["pre"][g]
        k, v = (torch.cat([a, _held(b, st["bt"][s], c + n)], 1) for a, b in zip(shared[g], (kc, vc)))
        for a in range(0, n, 512):
            m = min(n, a + 512) - a
            see = P + c + a + m
            x = q[at + a:at + a + m].view(m, hkv, hq // hkv, D).transpose(0, 1).reshape(hkv, -1, D)
            w = torch.matmul(x, k[:, :see].transpose(1, 2)).view(hkv, m, hq // hkv, see) * st["scale"]
            hide = torch.arange(see, device=DEV) > torch.arange(P + c + a, see, device=DEV).unsqueeze(1)
            w = w.masked_fill(hide[None, :, None, :], -math.inf)
            w = torch.exp(w - w.amax(-1, keepdim=True))
            w = w / w.sum(-1, keepdim=True)
            o = torch.matmul(w.view(hkv, -1, see), v[:, :see])
            out[at + a:at + a + m] = o.view(hkv, m, -1, D).transpose(0, 1).reshape(m, hq * D).to(BF16)
        at += n
    return [out, kc, vc]


def _plain_sample(st):
    x, n, V = st["x"], *st["x"].shape
    temp = st["temp"].double()
    greedy = temp <= 0
    v, order = torch.sort(x.float(), dim=-1, descending=True, stable=True)
    w = torch.exp((v.double() - v[:, :1].double()) / torch.where(greedy, 1.0, temp).unsqueeze(1))
    rank = torch.arange(V, device=DEV)
    k = torch.where((st["top_k"] > 0) & (st["top_k"] < V), st["top_k"], V).unsqueeze(1)
    w = torch.where(rank < k, w, 0.0)
    c = w.cumsum(-1)
    p = st["top_p"].double().unsqueeze(1)
    keep = (p >= 1) | (c - w < p * c[:, -1:])
    keep &= w >= st["min_p"].double().unsqueeze(1)
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    c = w.cumsum(-1)
    pick = (c <= st["u"].double().unsqueeze(1) * c[:, -1:]).sum(-1).clamp(max=V - 1)
    return torch.where(greedy, order[:, 0], pick)


def _plain_rows(x):
    """Codes (as fp32) and scales of rows."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    return torch.round(x * torch.where(top > 0, 127.0 / top, 0.0)), top / 127.0


def _plain_int8(st):
    q, s = _plain_rows(st["x"])
    wq, ws = st["w"]
    y = torch.matmul(q, wq.T) * (s * ws.T)
    return (y if st["bias"] is None else y + st["bias"].float()).to(BF16)


# ---------------------------------------------------------------------- run
def run(st):
    if not own:
        return {"share": _plain_share, "sample": _plain_sample, "int8": _plain_int8}[st["op"]](st)
    from swarmlora_amd import ops
    if st["op"] == "share":
        out = ops.prefix_attention(st["q"], st["k"], st["v"], st["kc"], st["vc"], st["pt"], st["plen"], st["bt"],
                                   st["lens"], st["pos"], st["cos_sin"], st["scale"], cu_groups=st["cg"],
                                   cu_seqlens=st["cu"])
        return [out, st["kc"], st["vc"]]
    if st["op"] == "sample":
        return ops.sample_tokens(st["x"], st["u"], st["temp"], st["top_k"], st["top_p"], st["min_p"])
    q, s = ops.int8_rows(st["x"])
    return ops.int8_matmul(q, s, st["w"], bias=st["bias"])


def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * 2 + 28), "flops": case["rows"] * case["vocab"] * 4}
    if case["op"] == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k + 4 * n + 2 * m * k + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    new, ctx, pre, size = _lens(case)
    hq, hkv, T = case["heads"], case["kv_heads"], sum(new)
    group = [g for g, n in enumerate(size) for _ in range(n)]
    seen = sum(n * (pre[g] + c) + n * (n + 1) // 2 for n, c, g in zip(new, ctx, group))
    # the caches read once, the new tokens' rows read, their keys and values stored, the result written
    return {"bytes": (sum(pre) + sum(ctx)) * hkv * 4 * D + T * ((hq + 2 * hkv) * 2 * D + hkv * 4 * D + hq * 2 * D + 2 * D + 8),
            "flops": seen * hq * 4 * D}


# -------------------------------------------------------------------- exact
def exact(case, seed):
    if case["op"] == "int8":
        return _exact_int8(case, seed)
    st = prepare(case, seed)
    return _exact_share(st) if case["op"] == "share" else _exact_sample(st)


def _exact_share(st):
    cs = st["cos_sin"][st["pos"]].double()
    turn = torch.complex(cs[:, :D // 2], cs[:, D // 2:]).unsqueeze(1)

    def rot(x):
        z = torch.complex(x[..., :D // 2].double(), x[..., D // 2:].double()) * turn
        return torch.cat([z.real, z.imag], -1)
    k, q = rot(st["k"]), rot(st["q"])
    kc, vc = st["kc"].double(), st["vc"].double()
    page, hq, hkv = kc.shape[1], q.shape[1], kc.shape[2]
    at = 0
    for s, (c, n) in enumerate(zip(st["ctx"], st["new"])):
        t = torch.arange(c, c + n, device=DEV)
        b = st["bt"][s].long()[t // page]
        kc[b, t % page], vc[b, t % page] = k[at:at + n], st["v"][at:at + n].double()
        at += n

    def held(cache, table, n, h):
        t = torch.arange(n, device=DEV)
        return cache[table.long()[t // page], t % page, h]
    out = torch.empty(st["T"], hq, D, dtype=torch.float64, device=DEV)
    for h in range(hkv):
        heads = range(h * hq // hkv, (h + 1) * hq // hkv)
        at, last = 0, None
        for s, (c, n, g) in enumerate(zip(st["ctx"], st["new"], st["group"])):
            if g != last:
                shared = [held(x, st["pt"][g], st["pre"][g], h) for x in (kc, vc)]
                last = g
            kh, vh = (torch.cat([a, held(x, st["bt"][s], c + n, h)]) for a, x in zip(shared, (kc, vc)))
            i = torch.arange(n, device=DEV)
            hide = torch.arange(len(kh), device=DEV) > (len(kh) - n + i).unsqueeze(1)
            for j in heads:
                sc = (q[at:at + n, j] @ kh.T) * st["scale"]
                out[at:at + n, j] = torch.softmax(sc.masked_fill(hide, -math.inf), -1) @ vh
            at += n
    return [out.flatten(1), kc, vc]


def _exact_sample(st):
    """One row after another, as the rule reads."""
    toks = []
    x, par = st["x"].double().cpu().numpy(), [st[k].double().tolist() for k in ("temp", "u", "top_k", "top_p", "min_p")]
    for row, t, u, k, p, m in zip(x, *par):
        order = np.lexsort((np.arange(len(row)), -row))
        if t <= 0:
            toks.append(int(order[0]))
            continue
        w = np.exp((row[order] - row[order[0]]) / t)
        count = int(k) if 0 < k < len(row) else len(row)
        if p < 1:
            c = np.cumsum(w[:count])
            count = int(np.searchsorted(c, p * c[-1], side="left")) + 1  # the first that reaches it
        count = max(1, min(count, int((w >= m).sum())))
        kept = np.zeros(len(row))
        kept[order[:count]] = w[:count]
        c = np.cumsum(kept)
        toks.append(int(np.searchsorted(c, u * c[-1], side="right")))
    return torch.tensor(toks)


def _exact_int8(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    w = _weight(case, gen).double()
    st = _activations(case, gen)

    def grid(a):
        top = a.abs().amax(1, keepdim=True)
        return torch.round(a * 127 / top.clamp(min=1e-300)), top / 127
    (q, s), (wq, ws) = grid(st["x"].double()), grid(w)
    y = (q @ wq.T) * s * ws.T
    return y if st["bias"] is None else y + st["bias"].double()
