"""GPU tests of the verification of drafted tokens (swl_verify_drafts_bf16)
against the rule in 64 bits on the CPU: tokens and counts have to be equal.
(A draw within 1e-13 of a border could differ; the seeds here have none.)"""

import math

import numpy as np
import pytest
import torch

from tests._util import BF16

pytestmark = pytest.mark.gpu


def _ops():
    from swarmlora_amd import ops
    return ops


def _first_largest(x):
    """First index of the largest logit, a NaN above all."""
    x = x.float().clone()
    if torch.isnan(x).any():
        return int(torch.isnan(x).int().argmax())
    return int((x == x.max()).int().argmax())


def _soft(x, t):
    x = x.double()
    e = torch.exp((x - x.max()) / t)
    return e / e.sum()


def rule(tgt, ids, u, u_last, temp, drf, new, max_drafts):
    toks, acc = [], []
    at = row = 0
    V = tgt.shape[1]
    for s, n in enumerate(new):
        t = float(temp[s])
        out, take = [], 0
        less = None
        for j in range(min(n, max_drafts)):
            x, d = tgt[row + j], int(ids[at + j])
            if t <= 0:
                if d != _first_largest(x):
                    break
            elif not 0 <= d < V:
                break
            else:
                p = _soft(x, t)
                q = _soft(drf[at + j], t) if drf is not None else torch.zeros(V, dtype=torch.float64).index_fill_(
                    0, torch.tensor([d]), 1.0)
                if not float(u[at + j]) * float(q[d]) < float(p[d]):
                    less = q if drf is not None else torch.where(torch.arange(V) == d, math.inf, 0.0).double()
                    break
            out.append(d)
            take += 1
        x = tgt[row + take]
        w = _soft(x, t) if t > 0 else torch.full((V,), math.nan)
        if less is not None:
            w = (w - less).clamp(min=0)
        c = np.cumsum(w.numpy())
        if t <= 0 or not c[-1] > 0:
            pick = _first_largest(x)
        else:
            want = float(u_last[s]) * c[-1]
            above = np.nonzero((c > want) & (w.numpy() > 0))[0]
            pick = int(above[0]) if len(above) else int(np.nonzero(w.numpy() > 0)[0][-1])
        toks.append(out + [pick] + [-1] * (max_drafts - take))
        acc.append(take)
        at += n
        row += n + 1
    return torch.tensor(toks), torch.tensor(acc, dtype=torch.int32)


def _case(seed, new, vocab, drafter, temps, near=0.7, pad=0):
    g = torch.Generator().manual_seed(seed)
    n, T = len(new), sum(new)
    tgt = 2.5 * torch.randn(T + n, vocab + pad, generator=g)
    rows = [r for s in range(n) for r in range(sum(new[:s]) + s, sum(new[:s]) + s + new[s])]
    drf = tgt[rows] + near * torch.randn(T, vocab + pad, generator=g)
    tgt, drf = tgt.to(BF16), drf.to(BF16)
    temp = torch.tensor([temps[s % len(temps)] for s in range(n)], dtype=torch.float32)
    seq = [s for s in range(n) for _ in range(new[s])]
    t = temp[seq].clamp(min=1e-3).unsqueeze(1)
    noise = -torch.log(-torch.log(torch.rand(T, vocab, generator=g).clamp(1e-20, 1 - 1e-7)))
    ids = (drf[:, :vocab].float() / t + noise).argmax(1) if T else torch.zeros(0, dtype=torch.int64)
    return {"tgt": tgt[:, :vocab], "drf": drf[:, :vocab] if drafter else None, "ids": ids, "temp": temp,
            "u": torch.rand(T, generator=g), "u_last": torch.rand(n, generator=g), "new": new}


def _run(c, dev, max_drafts=None):
    def put(x):  # (a padded row stays padded)
        if x is None:
            return None
        base = torch.empty(x.shape[0], x.stride(0), dtype=x.dtype, device=dev)
        base[:, :x.shape[1]] = x.to(dev)
        return base[:, :x.shape[1]]
    m = max(c["new"]) if max_drafts is None else max_drafts
    cu = torch.tensor([0] + list(c["new"])).cumsum(0).to(torch.int32).to(dev)
    tok, acc = _ops().verify_drafts(put(c["tgt"]), c["ids"].to(dev), c["u"].to(dev), c["u_last"].to(dev),
                                    c["temp"].to(dev), put(c["drf"]), cu_drafts=cu, max_drafts=m)
    torch.cuda.synchronize()
    return tok.cpu(), acc.cpu()


def _same(c, dev, max_drafts=None):
    m = max(c["new"]) if max_drafts is None else max_drafts
    got = _run(c, dev, max_drafts)
    want = rule(c["tgt"], c["ids"], c["u"], c["u_last"], c["temp"], c["drf"], c["new"], m)
    assert torch.equal(got[1], want[1]), (got[1], want[1])
    assert torch.equal(got[0], want[0]), (got[0], want[0])
    return got


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("new,vocab,temps,pad", [
    ([1], 1, [1.0], 0),
    ([0], 7, [0.5], 0),
    ([4], 32000, [0.8], 0),
    ([2, 0, 5, 1, 0, 3], 1001, [1.0, 0.0, 0.3], 0),          # rows that are not 16-byte aligned
    ([3, 1, 2], 2048, [0.7, 1.3], 40),                       # padded rows
    ([3] * 5, 2049, [1.0], 0),
    ([1, 5, 3, 2], 128256, [0.6, 1.0, 0.0], 0),
    ([2] * 70, 3000, [1.0, 0.9, 0.0, 2.0], 0),               # more than 64 sequences
    ([40, 17, 33], 500, [3.0, 8.0], 3),                      # more drafts than sixteen
    ([3] * 180, 16500, [0.9], 0),                            # rows of more than one slice
    ([1] * 1100, 4100, [0.8], 0),                            # a wave's share in two pieces, and in three
    ([1], 600001, [1.1], 0),
])
def test_tokens_and_counts_equal_the_rule(dev, new, vocab, temps, pad, drafter):
    for seed in range(3):
        _same(_case(seed + 10 * vocab, new, vocab, drafter, temps, near=0.3 if max(new) > 10 else 0.7, pad=pad), dev)


def test_uniform_form_and_fewer_drafts_than_given(dev):
    ops = _ops()
    c = _case(5, [4] * 6, 700, True, [0.9])
    tok, acc = ops.verify_drafts(c["tgt"].reshape(6, 5, 700).to(dev), c["ids"].view(6, 4).to(dev), c["u"].to(dev),
                                 c["u_last"].to(dev), c["temp"].to(dev), c["drf"].reshape(6, 4, 700).to(dev))
    want = _same(c, dev)
    assert torch.equal(tok.cpu(), want[0]) and torch.equal(acc.cpu(), want[1])
    _same(c, dev, max_drafts=2)   # later drafts do not count
    _same(c, dev, max_drafts=0)
    _same(c, dev, max_drafts=9)   # a wider output
    tok, acc = ops.verify_drafts(c["tgt"][:6].reshape(6, 1, 700).to(dev), torch.zeros(6, 0, dtype=torch.int64, device=dev),
                                 torch.zeros(0, device=dev), c["u_last"].to(dev), c["temp"].to(dev))
    assert tok.shape == (6, 1) and bool((acc == 0).all())


def test_greedy_ties_take_the_first(dev):
    new, V = [3, 2, 1], 5000
    c = _case(3, new, V, False, [0.0])
    for r in range(c["tgt"].shape[0]):
        c["tgt"][r, [100 + r, 4000]] = 30.0
    c["ids"] = torch.tensor([100, 101, 4000, 104, 105, 100])  # rows 0 1 2 3 | 4 5 6 | 7 8
    got = _same(c, dev)
    assert got[1].tolist() == [2, 2, 0]


def test_certain_tokens_masked_vocabularies_and_the_ends_of_u(dev):
    new, V = [2, 2, 2, 2], 3000
    c = _case(8, new, V, True, [1.0])
    for r in range(c["tgt"].shape[0]):  # a handful of tokens allowed
        keep = torch.randperm(V, generator=torch.Generator().manual_seed(r))[:5]
        m = torch.full((V,), -math.inf, dtype=BF16)
        m[keep] = c["tgt"][r, keep]
        c["tgt"][r] = m
    for u in (0.0, 1 - 2.0 ** -24, 1.0):
        c["u"][:], c["u_last"][:] = u, u
        _same(c, dev)
    # one token allowed: certain, and refused if it is not the draft
    c["tgt"][:] = -math.inf
    c["tgt"][:, 17] = 1.0
    c["ids"][:] = torch.tensor([17, 17, 17, 5, 5, 17, 17, 17])
    c["u"][:], c["u_last"][:] = 0.5, 0.5
    c["drf"] = None
    got = _same(c, dev)
    assert got[1].tolist() == [2, 1, 0, 2]
    # drafter and target agree wholly: accepted whatever u is
    c = _case(9, [3, 3], V, True, [0.7], near=0.0)
    c["u"][:] = 1 - 2.0 ** -24
    got = _same(c, dev)
    assert got[1].tolist() == [3, 3]


def test_rows_that_are_no_numbers_and_drafts_outside_the_vocabulary(dev):
    new, V = [2, 2, 2, 2, 2], 1500
    c = _case(12, new, V, True, [1.0])
    c["u"][:] = 0.0  # everything that can be is accepted
    c["tgt"][1, 700] = -math.nan               # row 1 of sequence 0 (a NaN of either sign)
    c["tgt"][1, 900] = math.nan
    c["tgt"][3, [9, 1200]] = math.inf          # row 0 of sequence 1
    c["tgt"][8] = -math.inf                    # row 2 of sequence 2
    c["ids"][6] = -1                           # sequence 3
    c["ids"][9] = V                            # sequence 4
    got = _same(c, dev)
    assert got[1].tolist() == [1, 0, 2, 0, 1]
    assert got[0][0, 1] == 700 and got[0][1, 0] == 9 and got[0][2, 2] == 0
    c["temp"][:] = 0.0
    _same(c, dev)
    # a NaN among masked logits, in a slice of nothing else
    new, V = [1, 1], 20000
    c = _case(13, new, V, True, [1.0])
    c["u"][:] = 0.0
    c["tgt"][:, 8:] = -math.inf
    c["tgt"][1, 15000] = math.nan
    c["tgt"][2, 15001] = math.nan
    c["ids"][:] = 3
    got = _same(c, dev)
    assert got[0].tolist() == [[3, 15000], [15001, -1]]


@pytest.mark.parametrize("temp", [3e38, math.inf])
def test_masked_tokens_stay_out_whatever_the_temperature(dev, temp):
    """-inf logits weigh 0 where the temperature makes all others alike."""
    ops, V = _ops(), 1003
    keep = torch.tensor([5, 17, 400, 1002])
    tgt = torch.full((2, V), -math.inf, dtype=BF16)
    tgt[:, keep] = torch.tensor([1.0, -3.0, 2.0, 0.5]).to(BF16)
    for u_last, want in ((0.1, 5), (0.3, 17), (0.6, 400), (0.9, 1002)):
        for drf in (None, tgt[:1].to(dev)):
            for d, u in ((400, 0.2), (3, 0.0)):  # accepted (p = 1 / 4); refused, and p is drawn from
                tok, acc = ops.verify_drafts(
                    tgt.to(dev).view(1, 2, V), torch.tensor([[d]], device=dev), torch.tensor([u], device=dev),
                    torch.tensor([u_last], device=dev), torch.tensor([temp], device=dev),
                    drf.view(1, 1, V) if drf is not None else None)
                if d == 400:
                    assert tok.tolist() == [[400, want]] and acc.tolist() == [1]
                elif drf is None:
                    assert tok.tolist() == [[want, -1]] and acc.tolist() == [0]
                else:  # p - q leaves nothing: the first largest logit
                    assert tok.tolist() == [[400, -1]] and acc.tolist() == [0]


@pytest.mark.parametrize("raised", [True, False])
def test_a_residual_far_smaller_than_the_rows(dev, raised):
    """Rows that differ in the draft and five tokens of little weight, so that
    their sums agree to under 3e-8 (raised: the residual is those five alone;
    lowered: every other token has a hundred-millionth of its weight left)."""
    n, V = 64, 20000
    g = torch.Generator().manual_seed(6)
    drf = (2.5 * torch.randn(V, generator=g)).to(BF16)
    few = [1500, 3333, 9001, 12345, 19000]  # slices of 2048: five of them
    drf[few] = torch.tensor([-6.0, -5.5, -6.5, -5.0, -7.0], dtype=BF16)
    tgt = drf.clone()
    drf[7], tgt[7] = -9.0, -10.0  # the draft
    tgt[few] = (drf[few].float() + (1.0 if raised else -1.0) * torch.tensor([0.25, 0.5, 0.25, 0.125, 0.5])).to(BF16)
    r = float(torch.exp(tgt.double()).sum() / torch.exp(drf.double()).sum()) - 1
    assert 5e-9 < abs(r) < 3e-8 and (r > 0) == raised
    c = {"tgt": tgt.expand(2 * n, V).contiguous(), "drf": drf.expand(n, V).contiguous(), "ids": torch.full((n,), 7),
         "temp": torch.ones(n), "u": torch.full((n,), 0.9), "u_last": (torch.arange(n) + 0.37) / n, "new": [1] * n}
    got = _same(c, dev)
    assert bool((got[1] == 0).all())
    seen = len(got[0][:, 0].unique())
    assert seen == 5 if raised else seen > 20


def test_drawn_tokens_follow_the_target(dev):
    """Over 20000 requests of the same two rows the first token (draft or
    drawn) has the target's distribution whatever the drafter's is: every
    frequency within 6 standard deviations of p (20 tokens: a chance of 4e-8)."""
    ops = _ops()
    n, V = 20000, 20
    g = torch.Generator().manual_seed(4)
    t, d = torch.randn(V, generator=g), torch.randn(V, generator=g)
    for drafter in (True, False):
        tgt = t.to(BF16).expand(n, 2, V).contiguous().to(dev)
        drf = d.to(BF16).expand(n, 1, V).contiguous().to(dev)
        ids = torch.multinomial(_soft(d.to(BF16), 0.8).float(), n, replacement=True, generator=g)
        u, ul = torch.rand(n, 1, generator=g), torch.rand(n, generator=g)
        tok, acc = ops.verify_drafts(tgt, ids.view(n, 1).to(dev), u.to(dev), ul.to(dev), torch.full((n,), 0.8, device=dev),
                                     drf if drafter else None)
        p = _soft(t.to(BF16), 0.8)
        f = torch.bincount(tok[:, 0].cpu(), minlength=V).double() / n
        assert bool(((f - p).abs() <= 6 * torch.sqrt(p * (1 - p) / n)).all())
        assert 0 < int(acc.sum()) < n


def test_captured_call_on_another_stream(dev):
    ops = _ops()
    new, V = [3, 1, 4], 32000
    c = _case(20, new, V, True, [0.9])
    cu = torch.tensor([0, 3, 4, 8], dtype=torch.int32, device=dev)
    d = {k: c[k].to(dev) for k in ("tgt", "drf", "ids", "u", "u_last", "temp")}

    def call():
        return ops.verify_drafts(d["tgt"], d["ids"], d["u"], d["u_last"], d["temp"], d["drf"], cu_drafts=cu, max_drafts=4)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tok, acc = call()
    for i in range(4):
        c = _case(30 + i, new, V, True, [0.9])
        for k in d:
            d[k].copy_(c[k])
        g.replay()
        torch.cuda.synchronize()
        want = rule(c["tgt"], c["ids"], c["u"], c["u_last"], c["temp"], c["drf"], new, 4)
        assert torch.equal(tok.cpu(), want[0]) and torch.equal(acc.cpu(), want[1])
        eager = call()
        assert torch.equal(eager[0], tok)


@pytest.mark.parametrize("drafter", [True, False])
def test_random_numbers_next_to_the_border(dev, drafter):
    """u so near to p / q that only 64 bits tell them apart (2^-15 to 2^-20 of
    it, either side; u itself is rounded by 2^-24)."""
    new, V = [5, 4, 20, 1, 3, 6], 4001
    c = _case(41, new, V, drafter, [0.9, 1.4], near=0.8)
    at = row = 0
    edge = [2.0 ** -15, -2.0 ** -17, 2.0 ** -20, -2.0 ** -15, -2.0 ** -20, 2.0 ** -17]
    near = 0
    for s, n in enumerate(new):
        t = float(c["temp"][s])
        for j in range(n):
            p, d = _soft(c["tgt"][row + j], t), int(c["ids"][at + j])
            q = float(_soft(c["drf"][at + j], t)[d]) if drafter else 1.0
            r = float(p[d]) / q
            if r < 0.95:
                # the last one refused; those before it accepted, however nearly
                c["u"][at + j] = r * (1 + (-abs(edge[(at + j) % 6]) if j < n - 1 else edge[s]))
                near += 1
        at += n
        row += n + 1
    got = _same(c, dev)
    assert near >= 12 and int(got[1].sum()) >= 12


@pytest.mark.parametrize("temp", [0.0, math.nan])
def test_zeros_of_either_sign_are_equal(dev, temp):
    """The first largest logit where -0 and +0 are the largest, -0 first: in one
    thread's logits, in one slice, and in two; greedy rows, and rows whose
    probabilities are no numbers (a temperature of NaN)."""
    places = [(1, 2), (9, 4000), (100, 20000), (8191, 8192)]
    V, n = 20001, 2 * len(places)
    tgt = torch.full((n, 2, V), -1.0, dtype=BF16)
    for i, (a, b) in enumerate(places):
        for j, (x, y) in enumerate(((-0.0, 0.0), (0.0, -0.0))):
            tgt[2 * i + j, :, a], tgt[2 * i + j, :, b] = x, y
    first = torch.tensor([a for a, _ in places for _ in range(2)])
    tok, acc = _ops().verify_drafts(tgt.to(dev), first.view(n, 1).to(dev), torch.zeros(n, 1, device=dev),
                                    torch.full((n,), 0.5, device=dev), torch.full((n,), temp, device=dev))
    if temp == 0.0:
        assert acc.tolist() == [1] * n and tok.cpu().tolist() == [[f, f] for f in first.tolist()]
    else:
        assert acc.tolist() == [0] * n and tok.cpu().tolist() == [[f, -1] for f in first.tolist()]


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("temp", [1e-4, 1e-6, 1e-30, 1e-40])
def test_temperatures_next_to_none(dev, temp, drafter):
    """Positive temperatures so small that a logit's exponent leaves 32 bits:
    all weight on the largest logits, shared where they tie."""
    new, V = [2, 3, 1, 2], 9000
    c = _case(17, new, V, drafter, [temp])
    c["temp"][:] = temp
    c["tgt"][:, 77] = -3e38
    c["tgt"][0, [5, 4000]] = 60.0   # a tie: half each
    c["tgt"][3, [6, 8999]] = 60.0
    c["tgt"][2, [7, 8]] = 60.0      # behind two accepted drafts
    c["ids"][0], c["ids"][2] = 5, 6
    c["u"][:] = 0.4
    if drafter:
        c["drf"][0, 5] = c["drf"][2, 6] = 90.0
        c["drf"][1, :] = c["tgt"][1, :]
    c["ids"][1] = int(c["tgt"][1].float().argmax())
    for u in (0.1, 0.7):
        c["u_last"][:] = u
        got = _same(c, dev)
        assert got[1][0] == 2 and got[0][0, 2] == (7 if u < 0.5 else 8)


@pytest.mark.parametrize("drafter", [True, False])
def test_drafts_behind_the_last_sequence_belong_to_none(dev, drafter):
    """Offsets that end before the drafts do: a captured call of fixed shapes
    whose offsets, drafts and temperatures change between replays."""
    ops, V, T, n = _ops(), 3001, 12, 4
    c = _case(50, [3] * n, V, drafter, [0.8])
    keys = [k for k in ("tgt", "drf", "ids", "u", "u_last", "temp") if c[k] is not None]
    d = {k: c[k].to(dev) for k in keys}
    cu = torch.zeros(n + 1, dtype=torch.int32, device=dev)

    def call():
        return ops.verify_drafts(d["tgt"], d["ids"], d["u"], d["u_last"], d["temp"], d.get("drf"), cu_drafts=cu, max_drafts=5)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, acc = call()
    for i, new in enumerate([[3, 3, 3, 3], [0, 5, 1, 2], [1, 0, 0, 0], [0, 0, 0, 0], [2, 4, 4, 2]]):
        c = _case(60 + i, new, V, drafter, [0.8, 0.0, 1.3])
        used = sum(new)
        for k, rows in (("tgt", used + n), ("drf", used), ("ids", used), ("u", used)):
            if k in d:
                d[k].fill_(math.nan if d[k].is_floating_point() else 7)
                d[k][:rows].copy_(c[k])
        d["u_last"].copy_(c["u_last"])
        d["temp"].copy_(c["temp"])
        cu.copy_(torch.tensor([0] + new).cumsum(0))
        graph.replay()
        torch.cuda.synchronize()
        want = rule(c["tgt"], c["ids"], c["u"], c["u_last"], c["temp"], c["drf"], new, 5)
        assert torch.equal(tok.cpu(), want[0]) and torch.equal(acc.cpu(), want[1])
        eager = call()
        assert torch.equal(eager[0], tok) and torch.equal(eager[1], acc)
