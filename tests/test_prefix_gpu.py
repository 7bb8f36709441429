"""GPU tests of attention over a shared prefix against its definition in 64
bits on the CPU."""

import math

import pytest
import torch

from tests import _prefix

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _case(seed, new, ctx, pre, size, hq=8, hkv=2, page=16, max_pos=4096, extra=0, spare=0):
    """Packed batch: new and cached tokens of the sequences, prefix lengths and
    sequence counts of the groups; `extra` token rows behind the last sequence."""
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    total = [max(c + n, 0) for c, n in zip(ctx, new)]
    need = [(n + page - 1) // page for n in pre + total]
    nb = sum(need) + 2
    perm = torch.randperm(nb, generator=g).to(torch.int32)
    w = max(need[:len(pre)] + [1])
    pt = torch.zeros(len(pre), w, dtype=torch.int32)
    bt = torch.zeros(len(new), max(need[len(pre):] + [1]) + spare, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        row = pt[i] if i < len(pre) else bt[i - len(pre)]
        row[:n] = perm[at:at + n]
        at += n
    T = sum(new) + extra
    kc, vc = (rn(nb, page, hkv, 128).to(BF16) for _ in range(2))
    qkv = rn(T, (hq + 2 * hkv) * 128).to(BF16)
    group = [i for i, n in enumerate(size) for _ in range(n)]
    pos = torch.cat([torch.arange(n) + c + (pre[group[s]] if s < len(group) else 0)
                     for s, (n, c) in enumerate(zip(new, ctx))] + [torch.zeros(extra, dtype=torch.int64)])
    ang = torch.outer(torch.arange(max_pos).double(), 10000.0 ** (-torch.arange(0, 128, 2).double() / 128))
    cum = lambda xs: torch.tensor([0] + list(torch.tensor(xs + [0]).cumsum(0)[:-1]), dtype=torch.int32)  # noqa: E731
    return dict(kc=kc, vc=vc, pt=pt, bt=bt, plens=torch.tensor(pre, dtype=torch.int32), cg=cum(size),
                lens=torch.tensor(ctx, dtype=torch.int32), cu=cum(new), qkv=qkv, pos=pos,
                cs=torch.cat([ang.cos(), ang.sin()], -1).to(BF16), hq=hq, hkv=hkv, scale=1 / math.sqrt(128))


def _views(c, qkv):
    hq, hkv, T = c["hq"], c["hkv"], qkv.shape[0]
    return (qkv[:, :hq * 128].view(T, hq, 128), qkv[:, hq * 128:(hq + hkv) * 128].view(T, hkv, 128),
            qkv[:, (hq + hkv) * 128:].view(T, hkv, 128))


def _run(c, dev, out=None):
    from swarmlora_amd import ops
    d = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    q, k, v = _views(c, d["qkv"])
    o = ops.prefix_attention(q, k, v, d["kc"], d["vc"], d["pt"], d["plens"], d["bt"], d["lens"], d["pos"], d["cs"],
                             c["scale"], cu_groups=d["cg"], cu_seqlens=d["cu"], out=out)
    assert torch.equal(d["qkv"].cpu().view(torch.int16), c["qkv"].view(torch.int16))
    return o, d


def _want(c):
    """(out, weight, k_cache, v_cache) by the definition; queries and keys are
    rounded to bf16 after the rotation, as they are held."""
    q, k, v = _views(c, c["qkv"])
    kc, vc = c["kc"].clone(), c["vc"].clone()
    rows = c["cs"][c["pos"].clamp(0, len(c["cs"]) - 1)]
    ok = ((c["pos"] >= 0) & (c["pos"] < len(c["cs"]))).view(-1, 1, 1)
    kr, qr = (torch.where(ok, _prefix.rotate(x, rows), x.double()).float().to(BF16) for x in (k, q))
    _prefix.store(kc, c["bt"], c["lens"], c["cu"], kr)
    _prefix.store(vc, c["bt"], c["lens"], c["cu"], v)
    o, w = _prefix.attend(qr, kc, vc, c["pt"], c["plens"], c["cg"], c["bt"], c["lens"], c["cu"], c["scale"])
    return o.flatten(1), w.flatten(1), kc, vc


def _check(c, dev):
    got, d = _run(c, dev)
    want, w, kc, vc = _want(c)
    n = int(c["cu"][-1])
    # rotations are fp32 sums of exact products, rounded to bf16: where fp32 and 64
    # bits round apart, one step of 2^-8 of the element
    kd = (d["kc"].cpu().double() - kc.double()).abs()
    assert bool((kd <= 2.0 ** -7 * kc.double().abs() + 1e-30).all()) and float((kd > 0).double().mean()) < 1e-3
    assert torch.equal(d["vc"].cpu().view(torch.int16), vc.view(torch.int16))
    # half a step of the result, and of the probabilities' bf16 (terms and sum: 2^-9
    # each way, 2^-8 together), as much again for a query or key rounded the other way
    off = (got.cpu().double()[:n] - want[:n]).abs()
    tol = 2.0 ** -8 * want[:n].abs() + 2.0 ** -7 * w[:n] + 1e-30
    bad = ~(off <= tol) & ~(torch.isnan(got.cpu()[:n]) & torch.isnan(want[:n]))
    assert not bool(bad.any()), (int(bad.sum()), float((off / tol).nan_to_num().max()))
    return got, d


@pytest.mark.parametrize("name,kw", [
    ("one token, one sequence", dict(new=[1], ctx=[0], pre=[1], size=[1])),
    ("no own tokens before", dict(new=[1, 1, 1], ctx=[0, 0, 0], pre=[70], size=[3])),
    ("prefix ends on a step", dict(new=[1, 1], ctx=[3, 64], pre=[128], size=[2])),
    ("prefix ends on a page", dict(new=[1] * 5, ctx=[0, 5, 16, 63, 64], pre=[48], size=[5])),
    ("long prefix in parts", dict(new=[1, 1, 1, 1], ctx=[7, 0, 300, 31], pre=[1531], size=[4])),
    ("empty prefix", dict(new=[1, 2], ctx=[9, 0], pre=[0], size=[2])),
    ("groups", dict(new=[1] * 7, ctx=[5, 0, 40, 9, 70, 1, 2], pre=[100, 0, 33], size=[3, 2, 2])),
    ("a group of nobody, a sequence of no group", dict(new=[1] * 4, ctx=[5, 0, 40, 9], pre=[100, 60, 33], size=[2, 0, 1])),
    ("drafts", dict(new=[1, 4, 6, 2, 0, 3], ctx=[5, 0, 40, 9, 3, 64], pre=[260], size=[6])),
    ("prompts beside tokens", dict(new=[1, 70, 1, 33, 31], ctx=[5, 0, 40, 9, 0], pre=[200], size=[5])),
    ("prompts alone", dict(new=[130, 64], ctx=[0, 17], pre=[90], size=[2])),
    ("long prompt without a prefix", dict(new=[150], ctx=[300], pre=[0], size=[1])),
    ("33 rows", dict(new=[1] * 11, ctx=[2] * 11, pre=[65], size=[11], hq=3, hkv=1)),
    ("129 rows", dict(new=[1] * 43, ctx=[2] * 43, pre=[65], size=[43], hq=3, hkv=1)),
    ("one head each", dict(new=[1, 3], ctx=[20, 1], pre=[81], size=[2], hq=4, hkv=4)),
    ("seven heads", dict(new=[1, 3], ctx=[20, 1], pre=[81], size=[2], hq=14, hkv=2)),
    ("many heads", dict(new=[1, 2], ctx=[20, 1], pre=[81], size=[2], hq=40, hkv=1)),
    ("pages of 1", dict(new=[1, 3], ctx=[20, 1], pre=[81], size=[2], page=1)),
    ("pages of 7", dict(new=[1, 30], ctx=[20, 1], pre=[81], size=[2], page=7)),
    ("pages of 24", dict(new=[1, 30], ctx=[20, 1], pre=[150], size=[2], page=24)),
    ("pages of 96", dict(new=[1, 30], ctx=[20, 1], pre=[150], size=[2], page=96)),
    ("rows behind", dict(new=[2, 1], ctx=[20, 1], pre=[81], size=[2], extra=3)),
    ("nothing before", dict(new=[3, 1], ctx=[-2, -1], pre=[0], size=[2], hq=4, hkv=2)),
    ("before the first own token", dict(new=[3, 1], ctx=[-2, -1], pre=[20], size=[2], hq=4, hkv=2)),
])
def test_against_the_definition(dev, name, kw):
    _check(_case(sum(map(ord, name)), **kw), dev)
