"""GPU tests of attention over the 4-bit cache where its work is cut otherwise
than by the least part: parts searched for so that all units run at once, as
many blocks as places, more sequences than lanes with long parts, cut blocks
beside whole ones, in the kernel for few rows, the one for many, and both at
once.  Every row is compared with the definition in 64 bits over the values read
back (which test_kv4_gpu.py compares byte by byte).

Tolerance as there: half a step of the result's bf16 (2^-8 of it), and relative
to A = sum p |v| the probabilities' rounding to bf16 (2^-8 of the terms and of
their sum, 2^-7 together at most; both are counted at their largest, so that the
fp32 scores' 2^-12 and sums' 2^-24 * sqrt(keys) have room beneath).
"""

import math

import pytest
import torch

from tests._util import BF16

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def _ops():
    from swarmlora_amd import ops
    return ops


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _prefix(counts):
    return _i32([0] + torch.tensor(counts).cumsum(0).tolist())


def _cache(total, hkv, page, g):
    """Pages with total[s] random tokens of every sequence, block tables of a
    random order."""
    need = [(t + page - 1) // page for t in total]
    perm = torch.randperm(sum(need), generator=g, device="cuda").to(torch.int32)
    bt = torch.full((len(total), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        bt[s, :n] = perm[at:at + n]
        at += n
    pages = _ops().kv4_pages(sum(need), page, hkv, "cuda")
    for s, n in enumerate(total):
        k = torch.randn(1, n, hkv, 128, generator=g, device="cuda").to(BF16)
        v = torch.randn(1, n, hkv, 128, generator=g, device="cuda").to(BF16)
        _ops().kv4_append(k, v, pages, bt[s:s + 1], _i32([0]))
    return pages, bt


def _check_sequence(out, q, k, v, ctx):
    """out, q [n, hq, 128] of a sequence's new tokens, k, v [keys, hkv, 128]."""
    n, hq, _ = q.shape
    hkv = k.shape[1]
    hide = torch.arange(k.shape[0], device="cuda") > ctx + torch.arange(n, device="cuda").unsqueeze(1)
    for j in range(hq):
        h = j * hkv // hq
        kh, vh = k[:, h].double().t().contiguous(), v[:, h].double().contiguous()
        p = torch.softmax(torch.matmul(q[:, j].double(), kh).mul_(SCALE).masked_fill_(hide, -math.inf), -1)
        want, a = torch.matmul(p, vh), torch.matmul(p, vh.abs())
        got = out[:, j].double()
        ok = (got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * a
        assert bool(ok.all()), f"head {j}: {int((~ok).sum())} off"


def _run(ctx, new, hq, hkv, page, hint=None, uniform=False):
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(len(ctx) * 1000 + max(ctx))
    total = [c + n for c, n in zip(ctx, new)]
    pages, bt = _cache(total, hkv, page, g)
    T, cu, lens = sum(new), _prefix(new), _i32(ctx)
    q = torch.randn(T, hq, 128, generator=g, device="cuda").mul_(2).to(BF16)
    out = torch.full((T, hq * 128), math.nan, dtype=BF16, device="cuda")
    if uniform:
        L = new[0]
        ops.kv4_attention(q.view(len(new), L, hq, 128), pages, bt, lens, SCALE, out=out.view(len(new), L, hq * 128))
    else:
        ops.kv4_attention(q, pages, bt, lens, SCALE, cu_seqlens=cu, max_q_len=hint, out=out)
    at = 0
    for s, n in enumerate(new):
        k, v = ops.kv4_read(pages, bt[s:s + 1], _i32([0]), total[s])
        if n:
            _check_sequence(out[at:at + n].view(n, hq, 128), q[at:at + n], k[0], v[0], ctx[s])
        at += n


def _spread(n, lo, hi, seed):
    return torch.randint(lo, hi, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("ctx,new,hq,hkv,page", [
    (_spread(32, 4000, 16000, 1), [1] * 32, 32, 8, 16),             # search, units of 16 rows
    (_spread(28, 2000, 12000, 2), [6] * 28, 32, 8, 32),             # search, units of 32
    ([16000] + [300] * 30, [1] * 31, 16, 8, 16),                    # one long sequence, the others whole
    (_spread(100, 500, 8000, 3), [1] * 100, 16, 8, 16),             # more sequences than lanes
    (_spread(90, 100, 6000, 4), _spread(90, 0, 9, 5), 32, 8, 48),   # the same, drafted tokens, some none
    (_spread(40, 3000, 6000, 6), [1] * 40, 160, 32, 16),            # as many blocks as places
    (_spread(70, 700, 1500, 7), [1] * 70, 160, 32, 64),             # both
])
@pytest.mark.parametrize("uniform", [False, True])
def test_few_rows(dev, ctx, new, hq, hkv, page, uniform):
    if uniform and len(set(new)) > 1:
        new = [3] * len(new)
    _run(ctx, new, hq, hkv, page, max(new), uniform)


@pytest.mark.parametrize("ctx,new,hq,hkv,page", [
    ([0], [4096], 32, 8, 16),                                       # as many blocks as places, none cut
    ([30000, 0], [128, 2048], 32, 8, 32),                           # the same, one sequence cut in many
    ([4000, 4000], [300, 300], 32, 8, 16),                          # search, cut in three
    ([4000] * 4, [300] * 4, 32, 8, 16),                             # search, left whole
    ([20000] + [600] * 80, [140] + [35] * 80, 16, 4, 16),           # more sequences than lanes
    ([9000, 100, 12000, 5000] + _spread(24, 200, 12000, 8), [512, 1, 512, 17] + [1] * 24, 32, 8, 32),  # mixed
    ([6000, 300] + _spread(80, 100, 4000, 9), [512, 700] + [2] * 80, 32, 8, 16),  # mixed, more sequences than lanes
])
def test_many_rows(dev, ctx, new, hq, hkv, page):
    _run(ctx, new, hq, hkv, page, max(new))
    if len(set(new)) == 1:
        _run(ctx, new, hq, hkv, page, None, True)


def test_hints_that_are_far_too_small(dev):
    """A call that takes the few-rows kernel whole by its hint: blocks of 16 rows,
    more of them than places, and cut ones."""
    _run([3000, 0, 9000], [200, 700, 3], 32, 8, 16, 1)
