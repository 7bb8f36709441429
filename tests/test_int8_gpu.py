"""GPU tests of products in 8-bit integers: codes and scales against the
definition in 64 bits, products against exact integer sums."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _randn(shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(BF16)


def codes(x):
    """(codes, scales) of rows, float64."""
    x = x.double()
    top = x.abs().amax(1, keepdim=True)
    bad = ~torch.isfinite(x).all(1, keepdim=True)
    q = torch.where(bad | (top == 0), 0.0, torch.round(torch.where(bad, 0.0, x) * 127 / torch.where(bad | (top == 0), 1.0, top)))
    return q, torch.where(bad, math.nan, top / 127)[:, 0]


def unpacked(w):
    """Codes of an Int8Weight by the layout's definition, float64 [n, k]."""
    d = w.data.cpu().view(torch.int8).double().view(-1, (w.k + 127) // 128 * 2, 4, 16, 16)  # tile, block, k / 16, row, k % 16
    full = d.permute(0, 3, 1, 2, 4).reshape(d.shape[0] * 16, -1)
    assert not full[w.n:].any() and not full[:, w.k:].any()
    return full[:w.n, :w.k]


def want(q, s, wq, ws, bias):
    y = (q @ wq.T) * s.view(-1, 1) * ws
    return y if bias is None else y + bias.double()


def check(y, q, s, wq, ws, bias):
    """Half a step of the result (bf16 has 8 significant bits: steps of 2^-7 from 1 to
    2, so 2^-8 of the result at most), of what is added to the bias three fp32
    roundings (sum, product of the scales, product: 2^-24 each) and of the result one
    more, together under 2^-22 of either."""
    t = want(q, s, wq, ws, bias)
    a = want(q, s, wq, ws, None)
    tol = (2.0 ** -8 + 2.0 ** -22) * t.abs() + 2.0 ** -22 * a.abs() + 1e-38
    off = (y.cpu().double() - t).abs()
    assert bool(((off <= tol) | (torch.isnan(y.cpu()) & torch.isnan(t))).all()), float((off / tol).nan_to_num().max())


@pytest.mark.parametrize("k", [1, 7, 16, 100, 4096, 14336, 16385, 40000])
def test_rows(dev, k):
    from swarmlora_amd import ops
    x = _randn((7, k), k)
    x[1] = 0
    x[2] *= 1e-38
    x[3] *= 1e30
    x[4, k // 2] = 127 * 2.0 ** -3  # codes that fall half way
    x[4, :k // 2] = (torch.arange(k // 2) % 255 - 127).to(BF16) * 2.0 ** -4
    x[5, 0] = float("inf")
    x[6, k - 1] = float("nan")
    q, s = ops.int8_rows(x.to(dev))
    wq, ws = codes(x)
    assert q.shape == (7, k) and q.dtype == torch.int8 and torch.equal(q.cpu().double(), wq)
    f = ws.float()
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(f))
    # one division in fp32, exact to half a step (and subnormal ones to half of the least)
    off = (s.cpu().double() - ws).abs().nan_to_num()
    assert bool((off <= 2.0 ** -24 * ws.nan_to_num() + 2.0 ** -150).all())


@pytest.mark.parametrize("m", [2 ** 22, 2 ** 22 + 5, 2 ** 24 + 5])
def test_more_rows_than_a_launch_has(dev, m):
    from swarmlora_amd import ops
    x = torch.randn(m, 1, generator=torch.Generator(dev).manual_seed(1), device=dev).to(BF16)
    q, s = ops.int8_rows(x)
    # (one division in fp32 on either side, exact to half a step)
    assert torch.equal(q, (127 * x.sign()).to(torch.int8))
    assert bool(((s.double() * 127 - x[:, 0].double().abs()).abs() <= 2.0 ** -24 * x[:, 0].double().abs()).all())


@pytest.mark.parametrize("n,k", [(130, 14336), (17, 40001), (28672, 130)])
def test_large_weight(dev, n, k):
    from swarmlora_amd import ops
    w = _randn((n, k), n + k)
    w[3] = 0
    p = ops.Int8Weight(w.to(dev))
    wq, ws = codes(w)
    assert torch.equal(unpacked(p), wq)
    assert bool(((p.scale.cpu().double() - ws).abs() <= 2.0 ** -24 * ws).all())


@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 129), (100, 1000), (130, 64)])
def test_weight(dev, n, k):
    from swarmlora_amd import ops
    big = _randn((n, k + 24), n + k)
    w = big[:, 5:5 + k]
    p = ops.Int8Weight(big.to(dev)[:, 5:5 + k])
    wq, ws = codes(w)
    assert p.shape == (n, k) and torch.equal(unpacked(p), wq)
    assert bool(((p.scale.cpu().double() - ws).abs() <= 2.0 ** -24 * ws).all())


SIZES = [(1, 1, 1), (1, 16, 128), (3, 17, 129), (16, 100, 4096), (17, 6144, 512), (28, 1031, 1000), (32, 64, 14336), (33, 48, 300),
         (64, 16400, 256), (65, 50, 700), (107, 4096, 1024), (128, 33, 96), (129, 33, 96), (200, 130, 5000), (300, 1001, 260),
         (513, 256, 2048), (860, 161, 3000), (2000, 5000, 130), (2325, 4864, 256), (4100, 2600, 130)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("with_bias", [False, True])
def test_product(dev, m, n, k, with_bias):
    from swarmlora_amd import ops
    x, w = _randn((m, k), m + k), _randn((n, k), n)
    bias = _randn((n,), 5, 10.0) if with_bias else None
    p = ops.Int8Weight(w.to(dev))
    q, s = ops.int8_rows(x.to(dev))
    y = ops.int8_matmul(q, s, p, None if bias is None else bias.to(dev))
    assert y.shape == (m, n) and y.dtype == BF16
    check(y, q.cpu().double(), s.cpu().double(), unpacked(p), p.scale.cpu().double(), bias)


# Every kernel that a call can take, over more steps of k than it has places for: 16, 32
# and 64 rows by one, two and four tiles of 16 channels a workgroup (waves of several
# steps each), tiles of 128 x 128 whole and with k split, tiles of 256 x 256.
LONG = [(16, 1000, 3000), (1, 12300, 1200), (28, 1031, 5000), (17, 6144, 2100), (28, 12300, 1200), (50, 700, 5000),
        (60, 4000, 3000), (64, 16400, 1200), (200, 3100, 1900), (1700, 1500, 1100), (2325, 4864, 1100), (2305, 4700, 3333)]


@pytest.mark.parametrize("m,n,k", LONG)
def test_product_of_many_steps(dev, m, n, k):
    """Codes that differ in every step, row and channel: a stage read too early or left
    from another one, or a swapped tile, has other sums."""
    from swarmlora_amd import ops
    p = ops.Int8Weight(_randn((n, k), n).to(dev))
    q, s = ops.int8_rows(_randn((m, k), m + k).to(dev))
    y = ops.int8_matmul(q, s, p)
    check(y, q.cpu().double(), s.cpu().double(), unpacked(p), p.scale.cpu().double(), None)


@pytest.mark.parametrize("m,n,k", [(5, 12300, 14336), (40, 12300, 8100), (40, 500, 14336), (300, 700, 14336), (2325, 4864, 4096)])
def test_largest_codes_by_channel_and_step(dev, m, n, k):
    """Codes of +-127 alone whose signs differ by channel, row and step of 64 k, so that
    sums lie between -k 127^2 and k 127^2, each another."""
    from swarmlora_amd import ops
    g = torch.Generator().manual_seed(m + n)
    sign = lambda *shape: 1 - 2 * torch.randint(0, 2, shape, generator=g)  # noqa: E731
    steps = (k + 63) // 64
    flip = torch.where(torch.rand(n, steps, generator=g) < torch.linspace(0, 1, n)[:, None], -1, 1)
    base = sign(k)
    wq = 127 * base * flip.repeat_interleave(64, 1)[:, :k]
    q = 127 * base * torch.where(torch.rand(m, steps, generator=g) < 0.1, -1, 1).repeat_interleave(64, 1)[:, :k]
    w = ops.Int8Weight((wq / 127).to(BF16).to(dev))
    assert torch.equal(unpacked(w), wq.double())
    room = torch.zeros(m, (k + 15) // 16 * 16, dtype=torch.int8)
    room[:, :k] = q
    s = torch.ones(m, device=dev)
    y = ops.int8_matmul(room.to(dev)[:, :k], s, w)
    check(y, q.double(), s.cpu().double(), wq.double(), w.scale.cpu().double(), None)


@pytest.mark.parametrize("m", [5, 40, 100, 300, 3000])
def test_largest_sums_are_exact(dev, m):
    """Codes of +-127 alone: 14336 * 127^2, and sums of 127 and -127 that leave 1."""
    from swarmlora_amd import ops
    k, n = 14336 if m < 3000 else 4096, 4200 if m == 3000 else 40
    q = torch.full((m, k), 127, dtype=torch.int8)
    q[1::2, ::2] = -127
    q[1::2, 0] = -126
    w = ops.Int8Weight(torch.ones(n, k, dtype=BF16, device=dev))
    s = torch.ones(m, device=dev)
    y = ops.int8_matmul(q.to(dev), s, w).cpu().double()
    t = (q.double().sum(1) * 127 / 127).view(-1, 1).expand(m, n)
    assert bool(((y - t).abs() <= (2.0 ** -8 + 2.0 ** -22) * t.abs()).all())


@pytest.mark.parametrize("m", [3, 20, 70, 600])
def test_longest_rows(dev, m):
    """131072 codes of -128 (made otherwise: rows have -127 at least) by 127, and of 127:
    sums within 32 bits by less than 1 %."""
    from swarmlora_amd import ops
    k, n = 131072, 40
    q = torch.full((m, k), -128, dtype=torch.int8)
    q[1::2] = 127
    w = ops.Int8Weight(torch.ones(n, k, dtype=BF16, device=dev))
    s = torch.ones(m, device=dev)
    check(ops.int8_matmul(q.to(dev), s, w), q.double(), s.cpu().double(), torch.full((n, k), 127.0).double(),
          w.scale.cpu().double(), None)


def test_views_and_strides(dev):
    from swarmlora_amd import ops
    m, n, k = 50, 70, 333
    big = _randn((m, k + 100), 1).to(dev)
    x = big[:, 3:3 + k]
    w = ops.Int8Weight(_randn((n, k), 2).to(dev))
    q, s = ops.int8_rows(x)
    q2, s2 = ops.int8_rows(x.contiguous())
    assert torch.equal(q, q2) and torch.equal(s, s2)
    y = ops.int8_matmul(q, s, w)
    wide = torch.full((m, 352), 77, dtype=torch.int8, device=dev)  # rows further apart, other bytes behind them
    wide[:, :k] = q
    out = torch.full((m, n + 6), 3.0, dtype=BF16, device=dev)
    got = ops.int8_matmul(wide[:, :k], s, w, out=out[:, :n])
    assert torch.equal(got, y) and bool((out[:, n:] == 3.0).all())
    for rows in (1, 20, 49):  # the same bits for any number of rows
        assert torch.equal(ops.int8_matmul(q[:rows], s[:rows], w), y[:rows])


def test_rows_that_are_no_numbers(dev):
    from swarmlora_amd import ops
    x = _randn((4, 256), 3)
    x[1, 9], x[2] = float("nan"), 0
    w = ops.Int8Weight(_randn((20, 256), 4).to(dev))
    q, s = ops.int8_rows(x.to(dev))
    y = ops.int8_matmul(q, s, w).cpu()
    assert bool(torch.isnan(y[1]).all()) and not bool(torch.isnan(y[[0, 2, 3]]).any()) and not bool(y[2].any())


@pytest.mark.parametrize("m,n,k", [(5, 600, 512), (200, 300, 4096), (600, 5000, 256)])
def test_captured_and_on_two_streams(dev, m, n, k):
    from swarmlora_amd import ops
    w = ops.Int8Weight(_randn((n, k), 1).to(dev))
    x = _randn((m, k), 2).to(dev)
    ops.int8_matmul(*ops.int8_rows(x), w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.int8_matmul(*ops.int8_rows(x), w)
    for seed in (3, 4, 5):
        x.copy_(_randn((m, k), seed))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.int8_matmul(*ops.int8_rows(x), w))
    xs = [_randn((m, k), 6 + i).to(dev) for i in range(2)]
    t = [ops.int8_matmul(*ops.int8_rows(a), w) for a in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.int8_matmul(*ops.int8_rows(xs[i]), w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, t[i]) for i in range(2) for a in got[i])


def test_refusals(dev):
    from swarmlora_amd import ops
    w = ops.Int8Weight(_randn((20, 100), 4).to(dev))
    q, s = torch.zeros(3, 100, dtype=torch.int8, device=dev), torch.ones(3, device=dev)
    with pytest.raises(ValueError, match="16-byte aligned"):
        ops.int8_matmul(q, s, w)  # rows 100 bytes apart
    with pytest.raises(ValueError, match="storage"):
        ops.int8_matmul(q[:1], s[:1], ops.Int8Weight(_randn((20, 100), 4).to(dev))) if q.untyped_storage().nbytes() < 112 else \
            ops.int8_matmul(torch.zeros(100, dtype=torch.int8, device=dev).view(1, 100), s[:1], w)
    good = torch.zeros(3, 112, dtype=torch.int8, device=dev)[:, :100]
    with pytest.raises(ValueError, match="one entry per row"):
        ops.int8_matmul(good, s[:2], w)
    with pytest.raises(ValueError, match="n elements"):
        ops.int8_matmul(good, s, w, bias=torch.zeros(19, dtype=BF16, device=dev))
    with pytest.raises(ValueError, match="expects q"):
        ops.int8_matmul(torch.zeros(3, 112, dtype=torch.int8, device=dev), s, w)
    with pytest.raises(ValueError, match="out must be"):
        ops.int8_matmul(good, s, w, out=torch.zeros(3, 19, dtype=BF16, device=dev))
    with pytest.raises(ValueError, match="unit column stride"):
        ops.int8_rows(torch.zeros(8, 8, dtype=BF16, device=dev).t())
    assert ops.int8_matmul(good[:0], s[:0], w).shape == (0, 20)
