"""GPU tests of the KV cache held in 4 bits: append with RoPE, read back and
attention, against the definition in 64 bits on the CPU (tests/_kv4.py).

Stored bytes are compared exactly: products of two bf16 are exact in fp32, so
the kernel's rotated keys carry one fp32 rounding, and a code differs from the
64-bit rule's only where that moves a value across a border (the seeds here
have none).  Attention, per element: half a step of the result's bf16 (2^-8 of
it), and relative to A = sum p |v|: the probabilities' rounding to bf16 (2^-8,
of the terms and of their sum 2^-7 together at most), fp32 scores (128 products of up
to 6 * 4 in units that sum to under 200 before the scale: 2^-24 * 200 * 4 twice,
under 2^-12) and sums over the keys (2^-24 * keys, under 2^-11 for 8192).
"""

import math

import pytest
import torch

from tests import _kv4
from tests._util import BF16, randn

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(128)


def _ops():
    from swarmlora_amd import ops
    return ops


def _tables(total, page, seed, spare=2):
    need = [(t + page - 1) // page for t in total]
    nb = sum(need) + spare
    perm = torch.randperm(nb, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    bt = torch.full((len(total), max(need) + 1), nb - 1 if spare == 0 else -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        bt[s, :n] = perm[at:at + n]
        at += n
    return bt, nb


def _wide(bt, wide=True):
    """The table with columns of no page, to 2^21 keys and more: a call that could
    be large by its shapes, which takes the kernels for many rows."""
    return torch.cat([bt, bt.new_full((bt.shape[0], (1 << 17) - bt.shape[1]), -1)], 1) if wide else bt


def _prefix(counts):
    return torch.tensor([0] + list(counts)).cumsum(0).to(torch.int32)


def _cos_sin(n):
    ang = torch.outer(torch.arange(n).double(), 500000.0 ** (-torch.arange(0, 128, 2).double() / 128))
    return torch.cat([ang.cos(), ang.sin()], -1).to(BF16)


def _filled(total, hkv, page, seed, missing=()):
    """A cache with `total[s]` random tokens per sequence, through the kernel
    (which the append tests compare byte by byte)."""
    bt, nb = _tables(total, page, seed)
    pages = _ops().kv4_pages(nb, page, hkv, "cuda")
    T = sum(total)
    k, v = randn((T, hkv, 128), seed + 1).cuda(), randn((T, hkv, 128), seed + 2).cuda()
    zero = torch.zeros(len(total), dtype=torch.int32, device="cuda")
    _ops().kv4_append(k, v, pages, bt.cuda(), zero, cu_seqlens=_prefix(total).cuda())
    for s, j in missing:
        bt[s, j] = -1
    return pages, bt


def _check(got, want, wt, slack):
    got = got.double().cpu().view_as(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    tol = 2.0 ** -8 * want.abs() + slack * wt + 1e-30
    bad = (got - want).abs() > tol
    bad &= ~torch.isnan(want)
    assert not bad.any(), f"{int(bad.sum())} off, worst {float(((got - want).abs() / tol).nan_to_num(0).max()):.2f} of the bound"


# ------------------------------------------------------------------ append
APPEND = [  # ctx, new, hq, hkv, page, rope, fused rows
    ([0], [1], 1, 1, 16, True, False),
    ([5, 0, 130], [1, 1, 1], 32, 8, 16, True, True),
    ([15, 16, 17, 0], [1, 33, 0, 70], 12, 4, 48, True, True),
    ([3, 40], [64, 5], 7, 1, 32, False, False),
    ([100, 7], [130, 257], 6, 3, 64, True, True),
]


@pytest.mark.parametrize("ctx,new,hq,hkv,page,rope,fused", APPEND)
def test_append_stores_the_nearest_codes(dev, ctx, new, hq, hkv, page, rope, fused):
    ops = _ops()
    T, extra = sum(new), 3  # rows behind the last sequence
    bt, nb = _tables([c + n for c, n in zip(ctx, new)], page, 5)
    rows = randn((T + extra, (hq + 2 * hkv) * 128), 7)
    rows[:, hq * 128:(hq + hkv) * 128] *= 3
    if fused:
        r = rows.to(dev)
        q, k, v = (x.unflatten(1, (-1, 128)) for x in r.split([hq * 128, hkv * 128, hkv * 128], 1))
    else:
        q, k, v = (x.contiguous().to(dev).unflatten(1, (-1, 128)) for x in rows.split([hq * 128, hkv * 128, hkv * 128], 1))
    seq = [s for s, n in enumerate(new) for _ in range(n)]
    pos = torch.tensor([c + i for c, n in zip(ctx, new) for i in range(n)] + [0] * extra)
    cs = _cos_sin(int(pos.max()) + 1)
    pages = torch.randint(0, 256, (nb, hkv, page // 16, 2176), generator=torch.Generator().manual_seed(9)).to(torch.uint8)
    dp = pages.to(dev)
    q_out = torch.full((T + extra, hq, 128), 7.0, dtype=BF16, device=dev)
    kept = k.clone()
    got = ops.kv4_append(k, v, dp, bt.to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev),
                         pos.to(dev) if rope else None, cs.to(dev) if rope else None, q=q,
                         cu_seqlens=_prefix(new).to(dev), q_out=q_out)
    assert got is q_out and torch.equal(k, kept)
    kk, vv, qq = k.cpu().double(), v.cpu().double(), q.cpu().double()
    if rope:
        kk, qq = _kv4.rotate(kk, cs[pos]), _kv4.rotate(qq, cs[pos])
    for t in range(T):
        _kv4.store(pages, bt, seq[t], int(pos[t]), kk[t], vv[t])
    assert torch.equal(dp.cpu(), pages)  # every byte, those of other tokens among them
    assert torch.equal(q_out[T:].cpu(), torch.full((extra, hq, 128), 7.0, dtype=BF16))
    d = (q_out[:T].cpu().double() - qq[:T]).abs()
    assert bool((d <= 2.0 ** -8 * qq[:T].abs() + 1e-30).all())


def test_append_uniform_in_place_and_unrotated_positions(dev):
    """[nseq, L, heads, 128] tokens without offsets; q rotated in place;
    positions outside the table leave their token unrotated."""
    ops = _ops()
    n, L, hq, hkv, page = 3, 5, 8, 2, 16
    ctx = torch.tensor([0, 14, 33], dtype=torch.int32)
    bt, nb = _tables([int(c) + L for c in ctx], page, 1)
    q, k, v = randn((n, L, hq, 128), 1), randn((n, L, hkv, 128), 2), randn((n, L, hkv, 128), 3)
    pos = (ctx.long().unsqueeze(1) + torch.arange(L)).reshape(-1)
    cs = _cos_sin(40)
    pos[2], pos[9] = -1, 40
    pages = ops.kv4_pages(nb, page, hkv, dev)
    dq = q.to(dev)
    out = ops.kv4_append(k.to(dev), v.to(dev), pages, bt.to(dev), ctx.to(dev), pos.to(dev), cs.to(dev), q=dq, q_out=dq)
    assert out is dq
    inside = ((pos >= 0) & (pos < 40)).view(n, L, 1, 1)
    rot = _kv4.rotate(q, cs[pos.clamp(0, 39)].view(n, L, 128))
    want = torch.where(inside, rot, q.double())
    assert bool(((dq.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-30).all())
    kr = torch.where(inside, _kv4.rotate(k, cs[pos.clamp(0, 39)].view(n, L, 128)), k.double())
    gk, gv = ops.kv4_read(pages, bt.to(dev), ctx.to(dev), L)
    assert torch.equal(gk.cpu().double(), _kv4.decode(*_kv4.encode(kr)))
    assert torch.equal(gv.cpu().double(), _kv4.decode(*_kv4.encode(v.double())))


def test_append_of_borders_extremes_and_nans(dev):
    """Ties, the borders between scales, zeros, the smallest and largest
    numbers, infinities and NaN, each in groups of its own."""
    ops = _ops()
    x = torch.zeros(20, 128)
    x[0, :16] = torch.tensor([4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, 6.0])
    x[1, :4] = torch.tensor([6.96875, 7.0, -7.0, 1.0])   # 7 moves the group to the next scale
    x[2, 0] = 6.96875
    x[3, 32] = 2.0 ** -120
    x[4, 64:96] = 2.0 ** -133                            # a subnormal bf16
    x[5, 0] = torch.finfo(BF16).max
    x[6, 0], x[6, 1] = 2.0 ** 127, -2.0 ** 120
    x[7, 0], x[8, 40], x[9, 127] = math.inf, -math.inf, math.nan
    x[10] = torch.randn(128, generator=torch.Generator().manual_seed(1)) * 1e-30
    x[11] = -0.0
    x[12] = torch.linspace(-8, 8, 128)
    x[13:] = torch.randn(7, 128, generator=torch.Generator().manual_seed(2)) * torch.logspace(-20, 20, 7).unsqueeze(1)
    x = x.to(BF16).unsqueeze(1)
    bt = torch.tensor([[1, 0]], dtype=torch.int32)
    pages = ops.kv4_pages(2, 16, 1, dev)
    ref = pages.cpu()
    ops.kv4_append(x.to(dev), x.flip(0).to(dev), pages, bt.to(dev), torch.zeros(1, dtype=torch.int32, device=dev),
                   cu_seqlens=torch.tensor([0, 20], dtype=torch.int32, device=dev))
    for t in range(20):
        _kv4.store(ref, bt, 0, t, x[t].double(), x[19 - t].double())
    same = pages.cpu() == ref
    # (codes of a NaN group mean nothing)
    k, v = ops.kv4_read(pages, bt.to(dev), torch.zeros(1, dtype=torch.int32, device=dev), 20)
    rk, rv, _ = _kv4.load(ref, bt, 0, 20)
    for got, want in ((k, rk), (v, rv)):
        got = got[0].cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))
    assert int((~same).sum()) <= 6 * 16  # six NaN groups of sixteen code bytes


def test_append_and_read_without_a_place(dev):
    """Tokens past the table or on a missing page are dropped and read as
    zeros; nothing else changes."""
    ops = _ops()
    bt = torch.tensor([[2, -1, 9], [0, 1, 3]], dtype=torch.int32)
    pages = torch.full((4, 2, 1, 2176), 17, dtype=torch.uint8, device=dev)
    k, v = randn((2, 48, 2, 128), 1), randn((2, 48, 2, 128), 2)
    lens = torch.tensor([0, 20], dtype=torch.int32)
    ops.kv4_append(k.to(dev), v.to(dev), pages, bt.to(dev), lens.to(dev))
    ref = torch.full((4, 2, 1, 2176), 17, dtype=torch.uint8)
    for s in range(2):
        for i in range(48):
            _kv4.store(ref, bt, s, int(lens[s]) + i, k[s, i].double(), v[s, i].double())
    assert torch.equal(pages.cpu(), ref)
    gk, gv = ops.kv4_read(pages, bt.to(dev), torch.zeros(2, dtype=torch.int32, device=dev), 60)
    for s in range(2):
        rk, rv, there = _kv4.load(ref, bt, s, 60)
        assert torch.equal(gk[s].cpu().double(), torch.where(there.view(-1, 1, 1), rk, 0.0).to(BF16).double())
        assert torch.equal(gv[s].cpu().double(), torch.where(there.view(-1, 1, 1), rv, 0.0).to(BF16).double())


def test_read_in_a_cache_past_32_bit_offsets(dev):
    ops = _ops()
    nb = 250_000  # 17408 bytes each: 4.35 GB
    pages = torch.empty(nb, 8, 1, 2176, dtype=torch.uint8, device=dev)
    bt = torch.tensor([[nb - 1, 3, nb - 2]], dtype=torch.int32)
    k, v, q = randn((1, 40, 8, 128), 1), randn((1, 40, 8, 128), 2), randn((1, 40, 8, 128), 3)
    zero = torch.zeros(1, dtype=torch.int32, device=dev)
    ops.kv4_append(k.to(dev), v.to(dev), pages, bt.to(dev), zero)
    gk, gv = ops.kv4_read(pages, bt.to(dev), zero, 40)
    assert torch.equal(gk.cpu().double(), _kv4.decode(*_kv4.encode(k.double())))
    assert torch.equal(gv.cpu().double(), _kv4.decode(*_kv4.encode(v.double())))
    out = ops.kv4_attention(q.to(dev), pages, bt.to(dev), zero, SCALE)
    few = torch.zeros(3, 8, 1, 2176, dtype=torch.uint8)
    fb = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    for i in range(40):
        _kv4.store(few, fb, 0, i, k[0, i].double(), v[0, i].double())
    want, wt = _kv4.attend(q[0], few, fb, [0], [0, 40], SCALE)
    _check(out, want, wt, 2.0 ** -7)


# --------------------------------------------------------------- attention
ATTEND = [  # ctx, new, hq, hkv, page
    ([0], [1], 1, 1, 16),                                     # one key
    ([0, 1, 15, 16, 31, 32, 33], [1] * 7, 8, 2, 16),          # around tiles and steps
    ([255, 256, 257, 511, 700, 1023], [1] * 6, 32, 8, 16),    # around parts
    ([5000, 3, 0, 2100], [1] * 4, 4, 1, 64),                  # many parts beside one
    ([40, 300], [1, 1], 7, 1, 48),                            # seven heads a kv head
    ([100, 80], [1, 1], 3, 3, 32),                            # a head each
    ([64, 900], [1, 1], 40, 2, 16),                           # twenty heads a kv head
    ([30, 500], [1, 1], 40, 1, 16),                           # forty, and seventy: a token's rows in several blocks
    ([30, 500], [1, 2], 70, 1, 16),
    ([12, 700, 0, 90], [3, 5, 2, 0], 32, 8, 16),              # drafted tokens, an empty sequence
    ([1500, 0, 33], [8, 1, 4], 16, 4, 32),
    ([0, 0, 0], [1, 70, 129], 8, 2, 16),                      # prompts
    ([37, 513], [200, 65], 8, 4, 48),                         # chunks behind cached tokens
    ([400, 2000, 10, 0, 77], [1, 150, 1, 33, 6], 16, 2, 16),  # a mixed batch
]


@pytest.mark.parametrize("ctx,new,hq,hkv,page", ATTEND)
def test_attention_matches_the_definition(dev, ctx, new, hq, hkv, page):
    ops = _ops()
    total = [c + n for c, n in zip(ctx, new)]
    pages, bt = _filled(total, hkv, page, 11)
    T, extra = sum(new), 2
    q = randn((T + extra, hq, 128), 3, 2.0)
    cu = _prefix(new)
    out = torch.full((T + extra, hq * 128), 5.0, dtype=BF16, device=dev)
    lens = torch.tensor(ctx, dtype=torch.int32)
    want, wt = _kv4.attend(q[:T], pages.cpu(), bt, ctx, cu.tolist(), SCALE)
    for hint, wide in ((max(new), False), (None, False), (max(new), True), (None, True)):
        out.fill_(5.0)
        got = ops.kv4_attention(q.to(dev), pages, _wide(bt, wide).to(dev), lens.to(dev), SCALE, cu_seqlens=cu.to(dev),
                                max_q_len=hint, out=out)
        assert got is out
        _check(out[:T], want, wt, 2.0 ** -7)
        assert bool((out[T:] == 5.0).all())


def test_more_sequences_than_lanes(dev):
    """150 sequences, some without new tokens, appended, read back and attended
    to in packed calls; the long ones behind the first 64."""
    ops = _ops()
    n, hq, hkv, page = 150, 4, 2, 16
    g = torch.Generator().manual_seed(9)
    ctx = torch.randint(0, 60, (n,), generator=g).tolist()
    new = torch.randint(0, 3, (n,), generator=g).tolist()
    ctx[70], ctx[140], new[70], new[130], new[149] = 1500, 700, 1, 50, 2
    pages, bt = _filled([c + m for c, m in zip(ctx, new)], hkv, page, 91)
    T, cu, lens = sum(new), _prefix(new), torch.tensor(ctx, dtype=torch.int32)
    k, v, q = randn((T, hkv, 128), 1), randn((T, hkv, 128), 2), randn((T, hq, 128), 3, 2.0)
    ops.kv4_append(k.to(dev), v.to(dev), pages, bt.to(dev), lens.to(dev), cu_seqlens=cu.to(dev))
    gk, gv = ops.kv4_read(pages, bt.to(dev), lens.to(dev), T, cu_seqlens=cu.to(dev))
    assert torch.equal(gk.cpu().double(), _kv4.decode(*_kv4.encode(k.double())))
    assert torch.equal(gv.cpu().double(), _kv4.decode(*_kv4.encode(v.double())))
    want, wt = _kv4.attend(q, pages.cpu(), bt, ctx, cu.tolist(), SCALE)
    for hint, wide in ((50, False), (None, True), (1, False)):
        out = ops.kv4_attention(q.to(dev), pages, _wide(bt, wide).to(dev), lens.to(dev), SCALE, cu_seqlens=cu.to(dev),
                                max_q_len=hint)
        _check(out, want, wt, 2.0 ** -7)


def test_one_token_of_any_stride(dev):
    """A lone token's own strides do not matter (an expanded or cut view)."""
    ops = _ops()
    pages, bt = _filled([20], 2, 16, 95)
    lens = torch.tensor([19], dtype=torch.int32, device=dev)
    q, k = randn((1, 1, 4, 128), 1).to(dev), randn((1, 1, 2, 128), 2).to(dev)
    a = pages.clone()
    ops.kv4_append(k, k, a, bt.to(dev), lens)
    b = pages.clone()
    odd = torch.as_strided(k, (1, 1, 2, 128), (1, 3, 128, 1))
    ops.kv4_append(odd, odd, b, bt.to(dev), lens)
    assert torch.equal(a, b)
    qo = torch.as_strided(q, (1, 1, 4, 128), (0, 5, 128, 1))
    assert torch.equal(ops.kv4_attention(qo, a, bt.to(dev), lens, SCALE), ops.kv4_attention(q, a, bt.to(dev), lens, SCALE))


@pytest.mark.parametrize("L", [1, 4, 33])
def test_attention_uniform_strided_and_a_wrong_hint(dev, L):
    """Queries in place in fused rows, [nseq, L, ..] without offsets; a
    max_q_len that is too small changes nothing but speed."""
    ops = _ops()
    n, hq, hkv, page = 5, 8, 2, 16
    ctx = [0, 10, 100, 300, 600]
    pages, bt = _filled([c + L for c in ctx], hkv, page, 21)
    rows = randn((n, L, (hq + 4) * 128), 4, 2.0)
    q = rows.to(dev)[..., :hq * 128].unflatten(-1, (hq, 128))
    lens = torch.tensor(ctx, dtype=torch.int32, device=dev)
    cu = [i * L for i in range(n + 1)]
    want, wt = _kv4.attend(q.cpu().reshape(n * L, hq, 128), pages.cpu(), bt, ctx, cu, SCALE)
    for wide in (False, True):
        _check(ops.kv4_attention(q, pages, _wide(bt, wide).to(dev), lens, SCALE), want, wt, 2.0 ** -7)
    packed = q.reshape(n * L, hq, 128)
    low = ops.kv4_attention(packed, pages, bt.to(dev), lens, SCALE, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=dev),
                            max_q_len=1)
    _check(low, want, wt, 2.0 ** -7)


def test_prompt_attention_whose_reference_is_left_far_behind(dev):
    """Rows of many: scores that grow along the keys by far more than 2^100,
    scores far below those of the first keys, and first pages that are missing
    in front of scores far below zero (the running maximum has to take over)."""
    ops = _ops()
    L, hq, hkv = 200, 4, 1
    for kind in range(3):
        bt, nb = _tables([L], 16, 61 + kind)
        k, v, q = randn((L, hkv, 128), 1), randn((L, hkv, 128), 2), randn((L, hq, 128), 3).abs()
        ramp = torch.linspace(0.0, 60.0, L).view(-1, 1, 1)
        sign = 1.0 if kind == 0 else -1.0
        k = (k.abs() * ramp * sign if kind < 2 else -k.abs() * 60).to(BF16)
        pages = ops.kv4_pages(nb, 16, hkv, "cuda")
        zero = torch.zeros(1, dtype=torch.int32, device=dev)
        cu = torch.tensor([0, L], dtype=torch.int32, device=dev)
        ops.kv4_append(k.to(dev), v.to(dev), pages, bt.to(dev), zero, cu_seqlens=cu)
        if kind == 2:
            bt[0, :3] = -1
        want, wt = _kv4.attend(q, pages.cpu(), bt, [0], [0, L], SCALE)
        for wide in (False, True):
            out = ops.kv4_attention(q.to(dev), pages, _wide(bt, wide).to(dev), zero, SCALE, cu_seqlens=cu)
            # sum |q k| up to 0.8 * 0.8 * 60 * 128 * scale = 440 before log2: its fp32 rounding, 2^-22 of it, moves p
            _check(out, want, wt, 2.0 ** -7 + 2.0 ** -22 * 440 * 8)


def test_attention_over_missing_pages_and_empty_rows(dev):
    ops = _ops()
    ctx, new = [300, 40, 20, 64], [1, 6, 40, 3]
    missing = [(0, 3), (0, 18), (1, 0), (1, 1), (1, 2), (2, 0), (2, 1), (3, 1)]
    pages, bt = _filled([c + n for c, n in zip(ctx, new)], 2, 16, 31, missing)
    bt[3, 2] = pages.shape[0] + 5  # past the pool
    q = randn((sum(new), 8, 128), 3, 2.0)
    cu = _prefix(new)
    want, wt = _kv4.attend(q, pages.cpu(), bt, ctx, cu.tolist(), SCALE)
    for wide in (False, True):
        out = ops.kv4_attention(q.to(dev), pages, _wide(bt, wide).to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev),
                                SCALE, cu_seqlens=cu.to(dev))
        _check(out, want, wt, 2.0 ** -7)
        assert bool((out[1:7] == 0).all())  # the second sequence has no page at all


def test_attention_lengths_past_the_table_or_negative(dev):
    """Keys past the table do not count; a sequence whose length is negative
    (an unused slot) sees what is left of it, or nothing."""
    ops = _ops()
    pages, bt = _filled([64, 64, 64], 1, 16, 41)
    bt = bt[:, :4].contiguous()
    ctx = [200, -1, -70]
    q = randn((3, 2, 4, 128), 3, 2.0)
    out = ops.kv4_attention(q.to(dev), pages, bt.to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev), SCALE)
    want, wt = _kv4.attend(q.view(6, 4, 128), pages.cpu(), bt, ctx, [0, 2, 4, 6], SCALE)
    _check(out, want, wt, 2.0 ** -7)
    assert bool((out[2] == 0).all()) and bool((out[1, 0] == 0).all())


@pytest.mark.parametrize("new", [[1, 1], [6, 3], [40, 100]])
def test_attention_nan_reaches_only_the_rows_that_see_it(dev, new):
    """NaN and infinities in keys, values and queries, and NaN groups in the
    places behind the last token."""
    ops = _ops()
    ctx = [70, 33]
    hkv, hq = 2, 8
    total = [c + n for c, n in zip(ctx, new)]
    bt, nb = _tables([t + 20 for t in total], 16, 51)
    pages = torch.full((nb, hkv, 1, 2176), 255, dtype=torch.uint8, device=dev)  # NaN everywhere
    k, v = randn((sum(total), hkv, 128), 1), randn((sum(total), hkv, 128), 2)
    k[total[0] - 1, 0, 5] = math.nan      # the last key of the first sequence, head 0
    v[total[0] - 1, 1, 40] = math.inf     # its value, head 1, dims 32..63
    v[total[0] + 20, 0, 100] = math.nan   # a cached value of the second, head 0, dims 96..127
    ops.kv4_append(k.to(dev), v.to(dev), pages, bt.to(dev), torch.zeros(2, dtype=torch.int32, device=dev),
                   cu_seqlens=_prefix(total).to(dev))
    q = randn((sum(new), hq, 128), 3, 2.0)
    q[0, 7, 3] = math.nan
    cu = _prefix(new)
    want, wt = _kv4.attend(q, pages.cpu(), bt, ctx, cu.tolist(), SCALE)
    for wide in (False, True):
        out = ops.kv4_attention(q.to(dev), pages, _wide(bt, wide).to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev),
                                SCALE, cu_seqlens=cu.to(dev))
        _check(out, want, wt.nan_to_num(0.0), 2.0 ** -7)
    assert bool(torch.isnan(want).any()) and not bool(torch.isnan(want).all())


def test_attention_of_large_and_tiny_scores(dev):
    """One key far above the rest, scores that grow along the keys, and all
    scores zero."""
    ops = _ops()
    ctx, hq, hkv = 600, 4, 1
    bt, nb = _tables([ctx + 1], 16, 61)
    k, v = randn((ctx + 1, hkv, 128), 1), randn((ctx + 1, hkv, 128), 2)
    k *= torch.linspace(0.1, 30, ctx + 1).view(-1, 1, 1).to(BF16)
    k[123] *= 50
    pages = ops.kv4_pages(nb, 16, hkv, dev)
    ops.kv4_append(k.to(dev), v.to(dev), pages, bt.to(dev), torch.zeros(1, dtype=torch.int32, device=dev),
                   cu_seqlens=torch.tensor([0, ctx + 1], dtype=torch.int32, device=dev))
    q = torch.stack([randn((4, 128), 3), randn((4, 128), 4, 1e-20), torch.zeros(4, 128, dtype=BF16)])
    q = torch.cat([q, (k[123, 0] / 50).expand(1, 4, 128).to(BF16)])
    for row in q:
        out = ops.kv4_attention(row.view(1, 1, 4, 128).to(dev), pages, bt.to(dev),
                                torch.tensor([ctx], dtype=torch.int32, device=dev), SCALE)
        want, wt = _kv4.attend(row.view(1, 4, 128), pages.cpu(), bt, [ctx], [0, 1], SCALE)
        # scores reach 1500 * 30 * 128: their fp32 rounding (2^-24 of sum |q k|) moves p by that much
        err = 2.0 ** -22 * float((row.double().abs() @ _kv4.load(pages.cpu(), bt, 0, ctx + 1)[0][:, 0].abs().T).max()) * SCALE
        _check(out, want, wt, 2.0 ** -7 + 4 * err)


# ---------------------------------------------------- together, as it is used
def test_chunks_tokens_and_drafts_of_one_cache(dev):
    """Two requests: their prompts in chunks, then single tokens and drafted
    ones, every pass appended and attended to, against one pass in 64 bits."""
    ops = _ops()
    hq, hkv, page = 8, 2, 16
    passes = [([0, 0], [50, 17]), ([50, 17], [33, 1]), ([83, 18], [1, 1]), ([84, 19], [4, 5]), ([86, 24], [1, 1])]
    total = [90, 30]
    bt, nb = _tables(total, page, 3)
    pages = ops.kv4_pages(nb, page, hkv, dev)
    ref = pages.cpu()
    cs = _cos_sin(100)
    for i, (ctx, new) in enumerate(passes):  # (the fifth pass takes two of the first request's drafts back)
        T = sum(new)
        rows = randn((T, (hq + 2 * hkv) * 128), 100 + i)
        q, k, v = (x.unflatten(1, (-1, 128)) for x in rows.split([hq * 128, hkv * 128, hkv * 128], 1))
        pos = torch.tensor([c + j for c, n in zip(ctx, new) for j in range(n)])
        seq = [s for s, n in enumerate(new) for _ in range(n)]
        cu, lens = _prefix(new), torch.tensor(ctx, dtype=torch.int32)
        dr = rows.to(dev)
        dq, dk, dv = (x.unflatten(1, (-1, 128)) for x in dr.split([hq * 128, hkv * 128, hkv * 128], 1))
        rot = ops.kv4_append(dk, dv, pages, bt.to(dev), lens.to(dev), pos.to(dev), cs.to(dev), q=dq, cu_seqlens=cu.to(dev))
        out = ops.kv4_attention(rot, pages, _wide(bt, i == 0).to(dev), lens.to(dev), SCALE, cu_seqlens=cu.to(dev),
                                max_q_len=max(new))
        kr = _kv4.rotate(k, cs[pos])
        for t in range(T):
            _kv4.store(ref, bt, seq[t], int(pos[t]), kr[t], v[t].double())
        assert torch.equal(pages.cpu(), ref)
        want, wt = _kv4.attend(rot.cpu(), ref, bt, ctx, cu.tolist(), SCALE)
        _check(out, want, wt, 2.0 ** -7)


def test_captured_step_follows_the_lengths(dev):
    """Append and attention captured once, replayed as the sequences grow, with
    eager calls between the replays; another graph of the same cache lives
    beside it."""
    ops = _ops()
    n, hq, hkv, page = 3, 8, 2, 16
    start = [0, 250, 511]
    pages, bt = _filled([s + 8 for s in start], hkv, page, 71)
    bt_d = bt.to(dev)
    lens = torch.tensor(start, dtype=torch.int32, device=dev)
    q, k, v = (randn((n, 1, h, 128), 5 + i).to(dev) for i, h in enumerate((hq, hkv, hkv)))
    out = torch.empty(n, 1, hq * 128, dtype=BF16, device=dev)

    def step():
        ops.kv4_append(k, v, pages, bt_d, lens)
        ops.kv4_attention(q, pages, bt_d, lens, SCALE, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
    for i in range(5):
        q.copy_(randn((n, 1, hq, 128), 50 + i))
        k.copy_(randn((n, 1, hkv, 128), 60 + i))
        v.copy_(randn((n, 1, hkv, 128), 70 + i))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got = out.clone()
        ctx = lens.tolist()
        want, wt = _kv4.attend(q.cpu().view(n, hq, 128), pages.cpu(), bt, ctx, list(range(n + 1)), SCALE)
        _check(got, want, wt, 2.0 ** -7)
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, got)
        lens += 1


@pytest.mark.parametrize("wide", [False, True])
def test_captured_packed_call_follows_the_offsets(dev, wide):
    """One captured call of append and attention over 80 token rows, replayed
    with other offsets and lengths: prompts beside single tokens, empty
    sequences, rows behind the last one left as they were."""
    ops = _ops()
    hq, hkv, page, T = 8, 2, 16, 80
    pages, bt = _filled([600, 400, 200], hkv, page, 73)
    bt_d = _wide(bt, wide).to(dev)
    q, k, v = (randn((T, h, 128), 5 + i).to(dev) for i, h in enumerate((hq, hkv, hkv)))
    cu, lens = (torch.zeros(n, dtype=torch.int32, device=dev) for n in (4, 3))
    out = torch.empty(T, hq * 128, dtype=BF16, device=dev)

    def step():
        ops.kv4_append(k, v, pages, bt_d, lens, cu_seqlens=cu)
        ops.kv4_attention(q, pages, bt_d, lens, SCALE, cu_seqlens=cu, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i, (new, ctx) in enumerate([([1, 70, 9], [500, 0, 100]), ([40, 0, 40], [0, 300, 160]), ([79, 1, 0], [510, 399, 7]),
                                    ([2, 2, 2], [3, 4, 5]), ([0, 0, 0], [1, 1, 1])]):
        q.copy_(randn((T, hq, 128), 50 + i, 2.0))
        k.copy_(randn((T, hkv, 128), 60 + i))
        cu.copy_(_prefix(new))
        lens.copy_(torch.tensor(ctx, dtype=torch.int32))
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        got, n = out.clone(), sum(new)
        assert bool((got[n:] == 5.0).all())
        want, wt = _kv4.attend(q[:n].cpu(), pages.cpu(), bt, ctx, _prefix(new).tolist(), SCALE)
        _check(got[:n], want, wt, 2.0 ** -7)
        step()
        assert torch.equal(out, got)


def test_two_streams_at_once(dev):
    """Calls of two streams share nothing: each has its own workspace."""
    ops = _ops()
    res = []
    cases = []
    for i in range(2):
        pages, bt = _filled([2000, 1500 + i, 900], 2, 16, 81 + i)
        q = randn((3, 1, 8, 128), 90 + i, 2.0)
        lens = torch.tensor([1999, 1499 + i, 899], dtype=torch.int32)
        cases.append((q.to(dev), pages, bt.to(dev), lens.to(dev)))
        res.append(_kv4.attend(q.view(3, 8, 128), pages.cpu(), bt, lens.tolist(), [0, 1, 2, 3], SCALE))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(ops.kv4_attention(*cases[i], SCALE))
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            assert torch.equal(o, outs[i][0])
        _check(outs[i][0], *res[i], 2.0 ** -7)


def test_worker_attention_over_a_cache_of_four_bits(dev):
    """WorkerBatchedOps.batch_flash_attention with a PagedKVCache4: prompts of
    two slots, then single tokens, one slot read back and freed."""
    from swarmlora_amd.worker.batched_ops import WorkerBatchedOps
    from swarmlora_amd.worker.paged_attention import PagedKVCache4
    hq, hkv, layers = 8, 2, 2
    kv = PagedKVCache4(layers, hkv, 128, 16, 3, 128, dev)
    cs = _cos_sin(128)
    refs = [p.cpu() for p in kv.pages]
    for step, q_len in enumerate([33, 1, 1]):
        sids = [2, 0]
        for s in sids:
            kv.ensure_blocks_for_length(s, kv.slot_seq_lens.get(s, 0) + q_len)
        lens = kv.get_seq_lens_tensor(sids)
        bt = kv.get_block_table_tensor(sids)
        pos = (lens.long().unsqueeze(1) + torch.arange(q_len, device=dev)).reshape(-1)
        meta = {"cache_seqlens": lens, "block_tables": bt, "positions": pos, "bufs_q": torch.empty(2, q_len, 0, device=dev)}
        for layer in range(layers):
            rows = {s: randn((1, q_len, (hq + 2 * hkv) * 128), 100 * step + 10 * layer + s) for s in sids}
            qkv = {s: r.to(dev).split([hq * 128, hkv * 128, hkv * 128], -1) for s, r in rows.items()}
            got = WorkerBatchedOps.batch_flash_attention(sids, qkv, kv, cs.to(dev), layer, hq, hkv, 128, meta)
            q, k, v = (torch.cat([rows[s][0] for s in sids]).split([hq * 128, hkv * 128, hkv * 128], -1)[i].unflatten(1, (-1, 128))
                       for i in range(3))
            at = pos.cpu()
            kr, qr = _kv4.rotate(k, cs[at]), _kv4.rotate(q, cs[at]).to(BF16)
            for t in range(2 * q_len):
                _kv4.store(refs[layer], bt.cpu(), t // q_len, int(at[t]), kr[t], v[t].double())
            assert torch.equal(kv.pages[layer].cpu(), refs[layer])
            want, wt = _kv4.attend(qr, refs[layer], bt.cpu(), lens.tolist(), [0, q_len, 2 * q_len], SCALE)
            _check(torch.cat([got[s] for s in sids]).view(2 * q_len, -1), want, wt, 2.0 ** -7)
        kv.advance_seq_lens(sids, q_len)
    k, v = kv.read(0, 1, 30)
    rk, rv, _ = _kv4.load(refs[1], kv.get_block_table_tensor([0]).cpu(), 0, 35)
    assert torch.equal(k.cpu().double(), rk[30:]) and torch.equal(v.cpu().double(), rv[30:])
    blocks = list(kv.slot_block_tables[2])
    kv.free_slot(2)
    for p in kv.pages:
        assert not bool(p[blocks].any()) and bool(p[kv.slot_block_tables[0]].any())


@pytest.mark.parametrize("ctx,new", [([700, 40], [1, 1]), ([300, 5], [6, 2]), ([60, 0], [150, 90])])
def test_attention_of_values_and_keys_of_every_scale(dev, ctx, new):
    """Value groups from 2^-110 to 2^100 beside one another, whole groups of zeros
    among them, and keys whose groups are up to 2^40 apart under queries that undo
    it."""
    ops = _ops()
    hq, hkv, page = 4, 2, 16
    total = [c + n for c, n in zip(ctx, new)]
    T = sum(total)
    g = torch.Generator().manual_seed(T)
    bt, nb = _tables(total, page, 17)
    v = randn((T, hkv, 128), 5).float().unflatten(-1, (4, 32))
    v = v * torch.exp2(torch.randint(-110, 101, (T, hkv, 4, 1), generator=g).float())
    v = (v * (torch.rand(T, hkv, 4, 1, generator=g) > 0.2)).flatten(-2).to(BF16)
    up = torch.exp2(torch.tensor([-20.0, 0.0, 20.0, 7.0])).repeat_interleave(32)
    k = (randn((T, hkv, 128), 6).float() * up).to(BF16)
    q = (randn((sum(new), hq, 128), 7).float() / up).to(BF16)
    pages = ops.kv4_pages(nb, page, hkv, dev)
    ops.kv4_append(k.to(dev), v.to(dev), pages, bt.to(dev), torch.zeros(2, dtype=torch.int32, device=dev),
                   cu_seqlens=_prefix(total).to(dev))
    # q's elements under 2^-13 of their row's largest are rounded by its operands (two fp8 numbers),
    # and these keys weigh them up again: the definition is taken over q as it is held
    big = q.double().abs().amax(-1, keepdim=True)
    s = torch.exp2(torch.floor(torch.log2(big)) - 7)
    held = _fp8_twice(q.double() / s) * s
    want, wt = _kv4.attend(held, pages.cpu(), bt, ctx, _prefix(new).tolist(), SCALE)
    for wide in (False, True):
        out = ops.kv4_attention(q.to(dev), pages, _wide(bt, wide).to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev),
                                SCALE, cu_seqlens=_prefix(new).to(dev))
        _check(out, want, wt, 2.0 ** -7)


def _fp8_twice(x):
    """x as an e4m3 number and what is left of it as another sixteenth of it,
    ties to even."""
    def e4m3(y):
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(y / step) * step
    hi = e4m3(x)
    return hi + e4m3((x - hi) * 16) / 16


def test_read_of_more_rows_than_the_sequences_have(dev):
    """Packed rows behind the last sequence hold anything; those before are
    what they are, empty sequences among them."""
    ops = _ops()
    pages, bt = _filled([40, 17, 90], 2, 16, 33)
    new, starts = [5, 0, 33], [30, 3, 50]
    k, v = ops.kv4_read(pages, bt.to(dev), torch.tensor(starts, dtype=torch.int32, device=dev), 100,
                        cu_seqlens=_prefix(new).to(dev))
    at = 0
    for s, n in enumerate(new):
        rk, rv, _ = _kv4.load(pages.cpu(), bt, s, starts[s] + n)
        assert torch.equal(k[at:at + n].cpu().double(), rk[starts[s]:]) and torch.equal(v[at:at + n].cpu().double(), rv[starts[s]:])
        at += n
