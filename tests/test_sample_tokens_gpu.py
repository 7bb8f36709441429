"""GPU tests of sampling from given random numbers, against the rule in 64 bits
(numpy, one row after another)."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def want_token(x, u, t, k=0, p=1.0, m=0.0):
    """The rule; x float64 [vocab]."""
    n = len(x)
    nan = np.isnan(x)
    key = np.where(nan, np.inf, x) + 0.0
    order = np.lexsort((np.arange(n), -key, ~nan))  # NaN above all
    top = x[order[0]]
    if not t > 0 or not np.isfinite(top):
        return int(order[0])
    with np.errstate(invalid="ignore"):
        w = np.exp((x[order] - top) / t)
    count = k if 0 < k < n else n
    if p < 1:
        c = np.cumsum(w[:count])
        count = int(np.searchsorted(c, p * c[-1], side="left")) + 1
    if m > 0:
        count = min(count, int((w >= m).sum()))
    count = max(count, 1)
    kept = np.zeros(n)
    kept[order[:count]] = w[:count]
    c = np.cumsum(kept)
    return min(int(np.searchsorted(c, u * c[-1], side="right")), int(np.nonzero(kept)[0][-1]))


def _f32(vals):
    return torch.tensor(vals, dtype=torch.float32)


def _check(dev, x, u, t, k=None, p=None, m=None, move=lambda a: a):
    from swarmlora_amd import ops
    n = x.shape[0]
    args = [_f32(u), _f32(t), None if k is None else torch.tensor(k, dtype=torch.int32), None if p is None else _f32(p),
            None if m is None else _f32(m)]
    got = ops.sample_tokens(move(x.to(dev)), *[None if a is None else a.to(dev) for a in args]).cpu()
    f = lambda a, i, d: d if a is None else a[i].double().item()  # noqa: E731
    want = [want_token(x[i].double().numpy(), f(args[0], i, 0), f(args[1], i, 0), int(f(args[2], i, 0)), f(args[3], i, 1.0),
                       f(args[4], i, 0.0)) for i in range(n)]
    assert got.tolist() == want
    return got


def _logits(n, V, seed, spikes=6):
    g = torch.Generator().manual_seed(seed)
    x = 2 * torch.randn(n, V, generator=g)
    for _ in range(spikes):
        x.scatter_add_(1, torch.randint(V, (n, 1), generator=g), 4 + 8 * torch.rand(n, 1, generator=g))
    return x.to(BF16), torch.rand(n, generator=g).tolist(), (0.3 + torch.rand(n, generator=g)).tolist()


FILTERS = [dict(), dict(k=1), dict(k=2), dict(k=50), dict(k=3000), dict(p=0.0), dict(p=1e-6), dict(p=0.5), dict(p=0.95),
           dict(p=0.9999), dict(m=0.05), dict(m=1.0), dict(m=1.5), dict(m=1e-12), dict(k=40, p=0.9), dict(k=500, p=0.99),
           dict(k=40, m=0.01), dict(p=0.9, m=0.02), dict(k=20, p=0.8, m=0.1), dict(k=-3, p=2.0, m=-1.0)]


@pytest.mark.parametrize("V", [1, 2, 7, 100, 8192, 8193, 32000])
@pytest.mark.parametrize("spikes", [0, 6])
def test_every_filter(dev, V, spikes):
    n = len(FILTERS) * 3
    x, u, t = _logits(n, V, V + spikes, spikes)
    f = [FILTERS[i % len(FILTERS)] for i in range(n)]
    _check(dev, x, u, t, [a.get("k", 0) for a in f], [a.get("p", 1.0) for a in f], [a.get("m", 0.0) for a in f])


def test_large_vocabulary(dev):
    n = len(FILTERS)
    x, u, t = _logits(n, 128256, 5)
    _check(dev, x, u, t, [a.get("k", 0) for a in FILTERS], [a.get("p", 1.0) for a in FILTERS],
           [a.get("m", 0.0) for a in FILTERS])
    x, u, t = _logits(2, 300000, 6)  # weights in fewer bits
    _check(dev, x, u, t, [0, 700], [0.9, 1.0], [0.0, 0.0])


@pytest.mark.parametrize("name", ["k", "p", "m", "none"])
def test_single_filters_without_the_others(dev, name):
    x, u, t = _logits(8, 5000, 9)
    _check(dev, x, u, t, **({} if name == "none" else {name: {"k": [30] * 8, "p": [0.9] * 8, "m": [0.05] * 8}[name]}))


def test_ties_go_to_the_lowest_index(dev):
    """Rows of few distinct logits: the border falls among equal ones."""
    g = torch.Generator().manual_seed(3)
    V, n = 9000, 24
    x = torch.randint(0, 3, (n, V), generator=g).to(BF16)
    x[4:8] = 1.0
    x[8:10] = torch.where(torch.randint(0, 2, (2, V), generator=g) == 0, 0.0, -0.0).to(BF16)
    u = torch.rand(n, generator=g).tolist()
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    k = [0, 1, 17, 300, 8999, 9000, 4000, 2, 5, 0] + [100 * i for i in range(14)]
    p = [1.0, 0.3, 0.9, 1.0, 0.5, 0.01, 1.0, 0.7, 1.0, 0.25] + [1.0, 0.5] * 7
    _check(dev, x, u, [0.5 + 0.1 * i for i in range(n)], k, p)


def test_rows_that_are_no_numbers_and_masks(dev):
    V = 8300
    x, u, t = _logits(12, V, 4)
    x[0, 77] = float("nan")
    x[1, 5000], x[1, 8200] = float("inf"), float("inf")
    x[2] = float("-inf")
    x[3, :] = float("-inf")
    x[3, 8299] = -3.0
    x[4, 10:] = float("-inf")  # ten tokens left
    x[5, ::2] = float("-inf")
    x[6] = torch.finfo(BF16).min
    x[7] = torch.finfo(BF16).min
    x[7, 100] = 1.0
    x[8] = torch.finfo(BF16).max
    x[9, 3] = torch.finfo(BF16).max
    x[10, 8292:] = float("nan")
    t[5], t[11] = 0.0, float("nan")
    k = [0, 3, 5, 40, 40, 0, 12, 5, 6, 0, 0, 0]
    _check(dev, x, u, t, k, [1.0, 0.9, 0.9, 0.9, 1.0, 1.0, 0.5, 0.9, 0.3, 0.9, 1.0, 1.0], [0.0, 0.1] * 6)


@pytest.mark.parametrize("t", [1e-30, 1e-3, 0.02, 5.0, 100.0, 1e30, float("inf")])
def test_temperatures(dev, t):
    x, u, _ = _logits(12, 20000, 8)
    _check(dev, x, u, [t] * 12, [0, 50, 0, 0, 900, 3] * 2, [1.0, 1.0, 0.9, 1.0, 0.99, 0.5] * 2, [0.0, 0.0, 0.0, 0.3, 0.0, 0.1] * 2)


@pytest.mark.parametrize("t", [1e37, 1e38, 3e38, float("inf")])
def test_logits_further_apart_than_the_largest_number(dev, t):
    # from -3.4e38 to 3.4e38: at these temperatures tokens of the lower half weigh
    # something too
    from swarmlora_amd import ops
    g = torch.Generator().manual_seed(13)
    big = torch.finfo(BF16).max
    x = ((2 * torch.rand(12, 9000, generator=g, dtype=torch.float64) - 1) * big).to(BF16)
    x[:, 100] = big
    x[6:, ::7] = -big
    x[9:, 1:8000] = float("-inf")
    u = ((torch.arange(12) + 0.5) / 12).tolist()
    k, p, m = [0, 8000, 0, 0, 5000, 30] * 2, [1.0, 1.0, 0.9, 1.0, 0.99, 0.5] * 2, [0.0, 0.0, 0.0, 0.3, 0.0, 0.1] * 2
    got = ops.sample_tokens(x.to(dev), *[_f32(a).to(dev) for a in (u, [t] * 12)], torch.tensor(k, dtype=torch.int32, device=dev),
                            _f32(p).to(dev), _f32(m).to(dev)).cpu()
    # an infinite temperature by 1e300: e^(-7e38 / 1e300) is 1 in 64 bits and e^(-inf /
    # 1e300) is 0, where -inf / inf is no number
    f = lambda a: float(_f32([a]))  # noqa: E731
    assert got.tolist() == [want_token(x[i].double().numpy(), f(u[i]), min(f(t), 1e300), k[i], f(p[i]), f(m[i]))
                            for i in range(12)]


def test_list_longer_than_its_room(dev):
    """A border among more tokens than are listed: all near one logit."""
    g = torch.Generator().manual_seed(2)
    x = (1 + 0.01 * torch.rand(6, 20000, generator=g)).to(BF16)
    x[3:] = torch.linspace(-1e-3, 1e-3, 20000)[torch.randperm(20000, generator=g)].to(BF16)
    _check(dev, x, torch.rand(6, generator=g).tolist(), [1.0] * 6, [7000, 0, 12345, 7000, 0, 5000],
           [1.0, 0.6, 0.5, 1.0, 0.31, 0.77])


def test_largest_vocabulary(dev):
    V = 1 << 21
    g = torch.Generator().manual_seed(21)
    x = torch.zeros(6, V, dtype=BF16)  # equal logits: all sums are whole numbers on either side
    x[3:, ::3] = float("-inf")
    _check(dev, x, torch.rand(6, generator=g).tolist(), [1.0] * 6, [0, 1000003, 0, 0, 700001, 5], [1.0, 1.0, 0.5, 1.0, 1.0, 1.0])


def test_most_rows(dev):
    from swarmlora_amd import ops
    n, V = 65535, 37
    g = torch.Generator(dev).manual_seed(22)
    x = torch.randn(n, V, generator=g, device=dev).to(BF16)
    u, t = torch.rand(n, generator=g, device=dev), 0.5 + torch.rand(n, generator=g, device=dev)
    k = torch.randint(0, V, (n,), generator=g, device=dev, dtype=torch.int32)
    got = ops.sample_tokens(x, u, t, k)
    for i in range(0, n, 8000):
        j = min(i + 8000, n)
        assert torch.equal(got[i:j], ops.sample_tokens(x[i:j], u[i:j].clone(), t[i:j].clone(), k[i:j].clone()))
    for i in (0, 1, 32767, 32768, 65533, 65534):
        assert int(got[i]) == want_token(x[i].cpu().double().numpy(), float(u[i]), float(t[i]), int(k[i]))


def test_strided_and_unaligned_rows(dev):
    x, u, t = _logits(9, 9001, 7)
    for pad in (1, 3, 8):
        _check(dev, x, u, t, [50] * 9, [0.9] * 9,
               move=lambda a: torch.cat([a.new_zeros(9, pad), a, a.new_zeros(9, pad)], 1)[:, pad:pad + 9001])


def test_distribution_follows_the_weights(dev):
    """Evenly spaced random numbers draw every token as often as its weight says."""
    from swarmlora_amd import ops
    N = 4096
    x = torch.tensor([[1.0, -2.0, 3.0, 0.5, 2.5, -1.0, 0.0, 1.5]]).to(BF16)
    u = (torch.arange(N) + 0.5) / N
    tok = ops.sample_tokens(x.to(dev).expand(N, 8).contiguous(), u.float().to(dev), torch.full((N,), 0.8, device=dev)).cpu()
    p = torch.softmax(x[0].double() / float(_f32([0.8])[0]), 0)
    assert bool((torch.bincount(tok, minlength=8).double() / N - p).abs().max() <= 1.0 / N)


def test_captured_call_follows_its_inputs(dev):
    from swarmlora_amd import ops
    n, V = 5, 40000
    x = torch.empty(n, V, dtype=BF16, device=dev)
    u, t = torch.empty(n, device=dev), torch.empty(n, device=dev)
    k, p, m = torch.empty(n, dtype=torch.int32, device=dev), torch.empty(n, device=dev), torch.empty(n, device=dev)

    def fill(seed):
        a, b, c = _logits(n, V, seed)
        x.copy_(a)
        u.copy_(_f32(b))
        t.copy_(_f32(c))
        k.copy_(torch.tensor([0, 50, 700, 0, seed + 1]))
        p.copy_(_f32([0.9, 1.0, 0.5, 1.0, 0.99]))
        m.copy_(_f32([0.0, 0.0, 0.1, 0.01 * seed, 0.0]))
        return [want_token(a[i].double().numpy(), u[i].double().item(), t[i].double().item(), int(k[i]), p[i].double().item(),
                           m[i].double().item()) for i in range(n)]
    fill(0)
    out = ops.sample_tokens(x, u, t, k, p, m)  # (loads the kernels)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.sample_tokens(x, u, t, k, p, m)
    for seed in range(1, 5):
        want = fill(seed)
        g.replay()
        torch.cuda.synchronize()
        assert out.tolist() == want
        assert torch.equal(out, ops.sample_tokens(x, u, t, k, p, m))


def test_two_streams_at_once(dev):
    from swarmlora_amd import ops
    sets = [[a.to(dev) if isinstance(a, torch.Tensor) else _f32(a).to(dev) for a in _logits(6, 30000, s)] for s in (1, 2)]
    p = torch.full((6,), 0.9, device=dev)
    want = [ops.sample_tokens(x, u, t, top_p=p) for x, u, t in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, (x, u, t)) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(s):
                got[i].append(ops.sample_tokens(x, u, t, top_p=p))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in (0, 1) for g in got[i])


def test_refusals(dev):
    from swarmlora_amd import ops
    x, u, t = torch.zeros(3, 10, dtype=BF16, device=dev), torch.zeros(3, device=dev), torch.ones(3, device=dev)
    with pytest.raises(ValueError, match="one entry per row"):
        ops.sample_tokens(x, u[:2], t)
    with pytest.raises(ValueError, match="contiguous"):
        ops.sample_tokens(x, torch.zeros(6, device=dev)[::2], t)
    with pytest.raises(TypeError, match="top_k must be torch.int32"):
        ops.sample_tokens(x, u, t, top_k=torch.zeros(3, dtype=torch.int64, device=dev))
    with pytest.raises(ValueError, match="unit column stride"):
        ops.sample_tokens(x.t(), torch.zeros(10, device=dev), torch.ones(10, device=dev))
    assert ops.sample_tokens(x[:0], u[:0], t[:0]).shape == (0,)
