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


@pytest.mark.parametrize("name,kw", [
    ("129 heads", dict(new=[1, 2], ctx=[20, 1], pre=[81], size=[2], hq=129, hkv=1)),
    ("200 heads of two", dict(new=[1, 2, 1], ctx=[20, 1, 300], pre=[700, 0], size=[2, 1], hq=400, hkv=2)),
    ("127 heads", dict(new=[1, 2, 0], ctx=[20, 1, 5], pre=[81], size=[3], hq=127, hkv=1)),
    ("128 heads behind nothing", dict(new=[1, 1], ctx=[20, 1], pre=[], size=[], hq=128, hkv=1)),
])
def test_more_heads_than_a_block_has_rows(dev, name, kw):
    _check(_case(sum(map(ord, name)), **kw), dev)


@pytest.mark.parametrize("name,kw", [
    ("many parts of a prefix", dict(new=[1, 1, 2], ctx=[20, 700, 1], pre=[20011], size=[3], max_pos=32768)),
    ("many sequences and groups", dict(new=[1] * 523, ctx=[i % 40 for i in range(523)], pre=[i % 70 for i in range(301)],
                                       size=[3 if i % 2 else 0 for i in range(301)], hq=2, hkv=1)),
    ("a wide table", dict(new=[1, 1], ctx=[20, 64], pre=[81], size=[2], spare=4000)),
    ("the longest step of few rows", dict(new=[1] * 8, ctx=[64, 0, 63, 65, 1, 127, 128, 129], pre=[64], size=[8], hq=16, hkv=4)),
])
def test_plans_against_the_definition(dev, name, kw):
    _check(_case(sum(map(ord, name)), **kw), dev)


def test_a_prompt_long_enough_to_be_cut_once_more(dev):
    # 207 blocks of rows x 63 steps, each counted twice, over 512 places: 51 steps
    # a place, more than the 32 that are cut
    c = _case(5, new=[3300], ctx=[0], pre=[700], size=[1], hq=8, hkv=1)
    got, d = _run(c, dev)
    q, k, v = _views(c, c["qkv"])
    rows = c["cs"][c["pos"]]
    qr, kr = (_prefix.rotate(x, rows).float().to(BF16) for x in (q, k))
    keys, vals = (torch.cat([_prefix.held(x, c["pt"][0], 700)[0], y.double()])[:, 0]
                  for x, y in ((c["kc"], kr), (c["vc"], v)))
    see = torch.arange(4000)[None] <= torch.arange(700, 4000)[:, None]
    for h in range(8):
        p = torch.softmax((qr[:, h].double() @ keys.T * c["scale"]).masked_fill(~see, -math.inf), -1)
        want, w = p @ vals, p @ vals.abs()
        # the tolerance of _check
        off = (got.cpu().double()[:, h * 128:(h + 1) * 128] - want).abs()
        assert bool((off <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * w + 1e-30).all()), h


MIXED = dict(new=[1, 4, 40, 2, 0, 1], ctx=[5, 0, 40, 9, 3, 130], pre=[260, 77], size=[4, 2])


def _seen(c):
    """Tokens of the cache [num_blocks, page] that some sequence sees or stores."""
    page = c["kc"].shape[1]
    m = torch.zeros(c["kc"].shape[:2], dtype=torch.bool)

    def mark(row, n):
        for p in range(max(n, 0)):
            if p // page < len(row) and 0 <= row[p // page] < len(m):
                m[row[p // page], p % page] = True

    for g in range(len(c["plens"])):
        mark(c["pt"][g].tolist(), int(c["plens"][g]))
    for s in range(len(c["lens"])):
        mark(c["bt"][s].tolist(), int(c["lens"][s] + c["cu"][s + 1] - c["cu"][s]))
    return m


@pytest.mark.parametrize("kw", [MIXED, dict(new=[1] * 5, ctx=[0, 5, 16, 63, 64], pre=[100], size=[5]),
                                dict(new=[140], ctx=[3], pre=[70], size=[1], page=96)])
def test_what_is_not_seen_does_not_matter(dev, kw):
    c = _case(31, **kw)
    want, _ = _run(c, dev)
    for fill in (math.nan, math.inf, -math.inf):
        d = dict(c, kc=c["kc"].clone(), vc=c["vc"].clone())
        d["kc"][~_seen(c)] = fill
        d["vc"][~_seen(c)] = fill
        got, _ = _run(d, dev)
        assert torch.equal(got.view(torch.int16), want.view(torch.int16)), fill


@pytest.mark.parametrize("kw", [MIXED, dict(new=[1] * 3, ctx=[40, 5, 16], pre=[100], size=[3])])
def test_pages_that_are_not_there_are_not_seen(dev, kw):
    c = _case(32, **kw)
    c["pt"][0, 1] = -1
    c["pt"][0, 4] = len(c["kc"])
    c["bt"][0, 0] = -7
    c["bt"][1, 0] = 2 ** 31 - 1
    c["bt"][2, 1] = len(c["kc"])
    _check(c, dev)


def test_a_sequence_none_of_whose_pages_are_there_has_zeros(dev):
    c = _case(33, new=[1, 3], ctx=[20, 1], pre=[81], size=[2])
    c["pt"][:] = -1
    c["bt"][1] = -1
    got, _ = _check(c, dev)
    assert not bool(got[1:].any())


@pytest.mark.parametrize("where", ["prefix", "own", "new"])
def test_not_a_number_reaches_those_that_see_it(dev, where):
    c = _case(34, **MIXED)
    v = _views(c, c["qkv"])[2]
    if where == "prefix":
        c["vc"][c["pt"][1, 1], 3, 0, 5] = math.nan
    elif where == "own":
        c["vc"][c["bt"][2, 0], 3, 1, 9] = math.nan
    else:
        v[3, 0, 17] = math.nan  # the third of the second sequence's four tokens
    got, _ = _check(c, dev)
    assert 0 < int(torch.isnan(got).sum()) < got.numel() // 8


def test_sums_that_leave_32_bits_are_done_again(dev):
    # sums of a few hundred values near 2^127 are no 32-bit numbers, their means are
    c = _case(35, **MIXED)
    c["vc"].mul_(0).add_(3e38)
    _views(c, c["qkv"])[2].mul_(0).add_(3e38)
    got, _ = _check(c, dev)
    assert bool(torch.isfinite(got).all())


def _check_unrotated(c, dev):
    """_check of a call without positions, whose queries and keys are what is given:
    fp32 and 64 bits see the same scores."""
    from swarmlora_amd import ops
    d = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    q, k, v = _views(c, c["qkv"])
    got = ops.prefix_attention(*_views(c, d["qkv"]), d["kc"], d["vc"], d["pt"], d["plens"], d["bt"], d["lens"], None, None,
                               c["scale"], cu_groups=d["cg"], cu_seqlens=d["cu"]).cpu()
    kc, vc = c["kc"].clone(), c["vc"].clone()
    _prefix.store(kc, c["bt"], c["lens"], c["cu"], k)
    _prefix.store(vc, c["bt"], c["lens"], c["cu"], v)
    o, w = _prefix.attend(q, kc, vc, c["pt"], c["plens"], c["cg"], c["bt"], c["lens"], c["cu"], c["scale"])
    o, w = o.flatten(1), w.flatten(1)
    ok = (got.double() - o).abs() <= 2.0 ** -8 * o.abs() + 2.0 ** -7 * w + 1e-30
    assert bool((ok | (torch.isnan(got) & torch.isnan(o))).all())
    return got, o


LARGE = [dict(new=[1, 1, 2, 1], ctx=[0, 1, 30, 5], pre=[0, 90], size=[2, 2]),
         dict(new=[1, 40, 33], ctx=[0, 2, 100], pre=[70], size=[3]),
         dict(new=[1, 1], ctx=[70, 3], pre=[1531], size=[2]),
         dict(new=[140], ctx=[3], pre=[70], size=[1], page=96)]


@pytest.mark.parametrize("kw", LARGE)
def test_scores_past_32_bits_of_an_exponent(dev, kw):
    # Scores near 2^40: a step of 32 bits there is thousands of powers of two.  The key of
    # the largest score is all of a row's result: the next one of any row is further
    # from it than 128 products' roundings, 128 * 2^-24 of the sum of their magnitudes.
    c = _case(46, **kw)
    hq, hkv = c["hq"], c["hkv"]
    c["qkv"][:, :(hq + hkv) * 128] *= 2.0 ** 18
    c["kc"] *= 2.0 ** 18
    q, k, _ = _views(c, c["qkv"])
    kc = c["kc"].clone()
    _prefix.store(kc, c["bt"], c["lens"], c["cu"], k)
    n = 0
    for s in range(len(kw["new"])):
        g = sum(s >= int(x) for x in c["cg"][1:])
        P, last = int(c["plens"][g]), int(c["lens"][s] + kw["new"][s])
        keys = torch.cat([_prefix.held(kc, c["pt"][g], P)[0], _prefix.held(kc, c["bt"][s], last)[0]])
        for i in range(kw["new"][s]):
            for h in range(hq):
                x = keys[:P + int(c["lens"][s]) + i + 1, h // (hq // hkv)]
                y = q[n + i, h].double()
                sc = (x @ y).sort(descending=True).values
                near = 128 * 2.0 ** -24 * float((x.abs() @ y.abs()).max())
                assert len(sc) == 1 or float(sc[0] - sc[1]) > 2 * near
        n += kw["new"][s]
    got, _ = _check_unrotated(c, dev)
    assert bool((got != 0).any(1).all())


@pytest.mark.parametrize("where", ["all", "prefix", "own", "first own", "prefix of values"])
@pytest.mark.parametrize("kw", LARGE)
def test_scores_of_minus_infinity(dev, kw, where):
    # q and k of dim 0 are 1 and, of some keys, -inf: rows that see no other keys have
    # 0 / 0, the others are as without these
    c = _case(47, **kw)
    q, k, v = _views(c, c["qkv"])
    q[..., 0] = 1
    if where in ("all", "prefix", "prefix of values"):
        for g in range(len(c["plens"])):
            for p in range(int(c["plens"][g])):
                c["kc"][c["pt"][g, p // c["kc"].shape[1]], p % c["kc"].shape[1], :, 0] = -math.inf
    if where == "prefix of values":  # 0 times an infinity is a NaN, whatever else the row sees
        c["vc"][c["pt"][-1, 0], 0, :, 7] = math.inf
    if where in ("all", "own", "first own"):
        for s in range(len(kw["new"])):
            for p in range(int(c["lens"][s])):
                c["kc"][c["bt"][s, p // c["kc"].shape[1]], p % c["kc"].shape[1], :, 0] = -math.inf
        (k if where != "first own" else k[:1])[..., 0] = -math.inf
    got, o = _check_unrotated(c, dev)
    assert torch.equal(torch.isnan(got), torch.isnan(o))
    assert where != "all" or bool(torch.isnan(got).all())


def test_without_new_keys_positions_or_offsets(dev):
    from swarmlora_amd import ops
    c = _case(36, new=[3] * 4, ctx=[5, 0, 40, 9], pre=[100], size=[4])
    d = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    q, k, v = _views(c, d["qkv"])
    packed = ops.prefix_attention(q, k, v, d["kc"], d["vc"], d["pt"], d["plens"], d["bt"], d["lens"], d["pos"], d["cs"],
                                  c["scale"], cu_seqlens=d["cu"])
    # [nseq, L]: the same call
    kc, vc = c["kc"].to(dev), c["vc"].to(dev)
    u = [t.view(4, 3, t.shape[1], 128) for t in (q, k, v)]
    even = ops.prefix_attention(*u, kc, vc, d["pt"], d["plens"], d["bt"], d["lens"], d["pos"], d["cs"], c["scale"])
    assert even.shape == (4, 3, 8 * 128) and torch.equal(even.flatten(0, 1), packed)
    assert torch.equal(kc, d["kc"]) and torch.equal(vc, d["vc"])
    # keys that are there already, queries rotated before
    qr = _prefix.rotate(_views(c, c["qkv"])[0], c["cs"][c["pos"]]).float().to(BF16)
    got = ops.prefix_attention(qr.to(dev), None, None, kc, vc, d["pt"], d["plens"], d["bt"], d["lens"], None, None,
                               c["scale"], cu_seqlens=d["cu"])
    assert torch.equal(kc, d["kc"]) and torch.equal(vc, d["vc"])
    o, w = _prefix.attend(qr, kc.cpu(), vc.cpu(), c["pt"], c["plens"], c["cg"], c["bt"], c["lens"], c["cu"], c["scale"])
    off = (got.cpu().double() - o.flatten(1)).abs()
    assert bool((off <= 2.0 ** -8 * o.flatten(1).abs() + 2.0 ** -7 * w.flatten(1) + 1e-30).all())


def test_no_prefix_at_all_is_paged_attention(dev):
    from swarmlora_amd import ops
    c = _case(37, new=[1] * 4, ctx=[5, 0, 140, 9], pre=[], size=[])
    d = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    q, k, v = (t.view(4, 1, t.shape[1], 128) for t in _views(c, d["qkv"]))
    kc, vc = c["kc"].to(dev), c["vc"].to(dev)
    got = ops.prefix_attention(q, k, v, kc, vc, d["bt"][:0, :0], d["plens"], d["bt"], d["lens"], d["pos"], d["cs"], c["scale"])
    want = ops.paged_attention(q, k, v, d["kc"], d["vc"], d["bt"], d["lens"], d["pos"], d["cs"], c["scale"])
    assert torch.equal(kc, d["kc"]) and torch.equal(vc, d["vc"])
    # both are off by half a step and their probabilities' roundings
    w = _want(c)[1].view(4, 1, -1)
    assert bool(((got.cpu() - want.cpu()).abs().double() <= 2.0 ** -7 * want.cpu().abs() + 2.0 ** -6 * w).all())


def test_sequences_before_the_first_group(dev):
    c = _case(38, new=[1, 2, 1, 1], ctx=[5, 0, 40, 9], pre=[100], size=[4])
    c["cg"] = torch.tensor([1, 3], dtype=torch.int32)
    _check(c, dev)


def test_offsets_that_overlap_stay_inside_what_is_there(dev):
    # [0, 4, 0, 4]: 8 tokens share their prefix by these offsets, but there are 4;
    # what such rows hold is not said, all else is as it was
    c = _case(44, new=[4, 0, 0], ctx=[20, 0, 20], pre=[81], size=[3])
    want, _ = _run(c, dev)
    bad = dict(c, cu=torch.tensor([0, 4, 0, 4], dtype=torch.int32))
    out = torch.full((8, 8 * 128), 7.0, dtype=BF16, device=dev)
    _, d = _run(bad, dev, out=out[:4])
    assert bool((out[4:] == 7).all())
    for n in ("pt", "bt", "plens", "lens", "cu", "cg", "cs", "pos"):
        assert torch.equal(d[n].cpu(), bad[n]), n
    assert torch.equal(_run(c, dev)[0], want)


def test_rows_before_the_first_sequence_are_left(dev):
    # rows 0 and 1 belong to nobody: stored, they would be the two tokens before those of
    # the first sequence
    c = _case(45, new=[5, 1], ctx=[20, 40], pre=[81], size=[2])
    c["cu"] = torch.tensor([2, 5, 6], dtype=torch.int32)
    out = torch.full((6, 8 * 128), 7.0, dtype=BF16, device=dev)
    got, d = _run(c, dev, out=out)
    want, w, kc, vc = _want(c)
    assert bool((got[:2] == 7).all())
    assert torch.equal(d["vc"].cpu().view(torch.int16), vc.view(torch.int16))
    off = (got.cpu().double() - want).abs()[2:]
    # the tolerance of _check
    assert bool((off <= 2.0 ** -8 * want[2:].abs() + 2.0 ** -7 * w[2:] + 1e-30).all())


def test_rows_behind_the_last_sequence_are_left(dev):
    c = _case(39, new=[2, 1, 30], ctx=[20, 1, 0], pre=[81], size=[3], extra=5)
    out = torch.full((38, 8 * 128), 7.0, dtype=BF16, device=dev)
    got, d = _run(c, dev, out=out)
    assert got.data_ptr() == out.data_ptr() and bool((out[33:] == 7).all())
    assert torch.equal(out[:33], _run(c, dev)[0][:33])


def test_caches_past_four_gigabytes(dev):
    c = _case(40, new=[1, 2, 150], ctx=[30, 0, 17], pre=[100], size=[3])
    want, d = _run(c, dev)
    # 16 tokens of 2 heads are 8 KiB: 600000 pages are 4.9 GB a cache
    far = 600000 - len(c["kc"])
    big = dict(d)
    for n in ("kc", "vc"):
        big[n] = torch.empty(600000, *c["kc"].shape[1:], dtype=BF16, device=dev)
        big[n][far:] = c[n].to(dev)
    for n in ("pt", "bt"):
        big[n] = d[n] + far
    assert torch.equal(_run_there(big), want)
    assert torch.equal(big["kc"][far:], d["kc"]) and torch.equal(big["vc"][far:], d["vc"])


def _run_there(d, out=None):
    """The call on what is on the device already, in place."""
    from swarmlora_amd import ops
    q, k, v = _views(d, d["qkv"])
    return ops.prefix_attention(q, k, v, d["kc"], d["vc"], d["pt"], d["plens"], d["bt"], d["lens"], d["pos"], d["cs"],
                                d["scale"], cu_groups=d["cg"], cu_seqlens=d["cu"], out=out)


def test_captured_calls_follow_lengths_and_tables(dev):
    """Two graphs of calls, each replayed several times with other lengths, tables
    and groups behind the same addresses, eager calls between them."""
    cases = [_case(50 + i, new=n, ctx=c, pre=p, size=z) for i, (n, c, p, z) in enumerate([
        ([1, 1, 1, 1], [5, 0, 40, 9], [100, 0], [3, 1]), ([1, 1, 1, 1], [6, 1, 300, 0], [0, 999], [1, 3]),
        ([1, 1, 1, 1], [0, 0, 0, 0], [17, 64], [2, 2]), ([4, 0, 0, 0], [3, 1, 1, 1], [64, 640], [4, 0])])]
    # buffers as large as the largest case's
    size = {n: [max(c[n].shape[i] for c in cases) for i in range(c0.dim())]
            for n, c0 in cases[0].items() if isinstance(c0, torch.Tensor)}

    def load(d, c):
        for n, s in size.items():
            t = torch.zeros(s, dtype=c[n].dtype)
            t[tuple(slice(0, x) for x in c[n].shape)] = c[n]
            d[n].copy_(t)

    state = [dict({n: torch.zeros(s, dtype=cases[0][n].dtype, device=dev) for n, s in size.items()}, hq=8, hkv=2,
                  scale=cases[0]["scale"]) for _ in range(2)]
    graphs, outs = [], []
    for d in state:
        load(d, cases[0])
        _run_there(d)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_run_there(d))
        graphs.append(g)
    for i in (1, 2, 0, 3, 1):
        for d, j in zip(state, (i, (i + 1) % 4)):
            load(d, cases[j])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o, j in zip(outs, (i, (i + 1) % 4)):
            want, _ = _run(cases[j], dev)
            assert torch.equal(o, want), (i, j)


def test_two_streams_at_once(dev):
    cases = [_case(60 + i, **MIXED) for i in range(2)]
    want = [_run(c, dev)[0] for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    state = [[{k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()} for _ in range(4)] for c in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for r in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_run_there(state[i][r]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])


def test_new_keys_as_they_are_and_queries_alone_rotated(dev):
    from swarmlora_amd import ops
    c = _case(41, new=[3, 1, 40], ctx=[5, 0, 9], pre=[100], size=[3])
    d = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    q, k, v = _views(c, c["qkv"])
    kc, vc = c["kc"].clone(), c["vc"].clone()
    _prefix.store(kc, c["bt"], c["lens"], c["cu"], k)
    _prefix.store(vc, c["bt"], c["lens"], c["cu"], v)
    dq, dk, dv = _views(c, d["qkv"])
    call = lambda k, v, pos, cs: ops.prefix_attention(  # noqa: E731
        dq, k, v, d["kc"], d["vc"], d["pt"], d["plens"], d["bt"], d["lens"], pos, cs, c["scale"], cu_groups=d["cg"],
        cu_seqlens=d["cu"])
    for args, qr in (((dk, dv, None, None), q),
                     ((None, None, d["pos"], d["cs"]), _prefix.rotate(q, c["cs"][c["pos"]]).float().to(BF16))):
        got = call(*args)
        assert torch.equal(d["kc"].cpu(), kc) and torch.equal(d["vc"].cpu(), vc)
        o, w = _prefix.attend(qr, kc, vc, c["pt"], c["plens"], c["cg"], c["bt"], c["lens"], c["cu"], c["scale"])
        off = (got.cpu().double() - o.flatten(1)).abs()
        # the tolerance of _check
        assert bool((off <= 2.0 ** -8 * o.flatten(1).abs() + 2.0 ** -7 * w.flatten(1) + 1e-30).all())


def test_refusals_of_the_front_end(dev):
    from swarmlora_amd import ops
    c = _case(42, new=[1, 2], ctx=[5, 0], pre=[30, 20], size=[1, 1])
    d = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    q, k, v = _views(c, d["qkv"])
    base = dict(q=q, k=k, v=v, k_cache=d["kc"], v_cache=d["vc"], prefix_table=d["pt"], prefix_lens=d["plens"],
                block_table=d["bt"], cache_seqlens=d["lens"], positions=d["pos"], cos_sin=d["cs"],
                softmax_scale=c["scale"], cu_groups=d["cg"], cu_seqlens=d["cu"])
    for kw, text in ((dict(cu_groups=None), "cu_groups"), (dict(k=None), "go together"), (dict(positions=None), "go together"),
                     (dict(cu_groups=d["cg"][:2]), "ngroups"), (dict(prefix_lens=d["plens"][:1]), "ngroups"),
                     (dict(block_table=d["bt"][:1]), "nseq"), (dict(k=k[:2]), "same tokens"),
                     (dict(v_cache=d["vc"][:1]), "contiguous"), (dict(positions=d["pos"][:2]), "positions"),
                     (dict(block_table=d["bt"].long()), "block_table"), (dict(out=d["qkv"][:, :1024]), "out"),
                     (dict(q=q[:, :7]), "multiple"), (dict(cache_seqlens=c["lens"]), "cache_seqlens")):
        with pytest.raises((ValueError, TypeError, RuntimeError), match=text):
            ops.prefix_attention(**{**base, **kw})
    with pytest.raises(RuntimeError, match="scale"):
        ops.prefix_attention(**{**base, "softmax_scale": 0.0})
