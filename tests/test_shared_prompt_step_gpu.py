"""GPU test of a decode step for sequences that go on from shared prompts, built
of products in 8-bit integers, attention over the shared prefixes and sampling
from given random numbers: eager and as a replayed graph, every operator against
its definition on what the one before it left."""

from types import SimpleNamespace

import pytest
import torch

from tests import test_int8_gpu as int8
from tests import test_prefix_gpu as prefix
from tests.test_sample_tokens_gpu import want_token

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HIDDEN, HQ, HKV, VOCAB = 264, 8, 2, 1003


def _state(dev, drafts):
    """Sequences of two shared prompts; `drafts`: several tokens of one of them a step."""
    from swarmlora_amd import ops
    new = [1, 1, 3, 1, 2, 1] if drafts else [1] * 6
    # (room for the tokens of 5 steps)
    c = prefix._case(70 + drafts, new=[5 * n for n in new], ctx=[5, 0, 40, 9, 31, 130], pre=[300, 77], size=[4, 2])
    n = sum(new)
    s = SimpleNamespace(ops=ops, n=n, **{k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in c.items()
                                         if k not in ("qkv", "cu", "pos")})
    s.new = torch.tensor(new, dtype=torch.int32)
    s.cu = torch.cat([torch.zeros(1, dtype=torch.int32), s.new.cumsum(0).int()]).to(dev)
    g = torch.Generator().manual_seed(71)
    first = [int(c["lens"][i]) + (300 if i < 4 else 77) for i in range(6)]
    s.pos = torch.cat([torch.arange(k) + f for k, f in zip(new, first)]).to(dev)
    s.step_of = torch.repeat_interleave(s.new, s.new.long()).long().to(dev)
    s.embed = torch.randn(VOCAB, HIDDEN, generator=g).to(BF16).to(dev)
    w = lambda o, i, std: torch.randn(o, i, generator=g).mul(std).to(BF16).to(dev)  # noqa: E731
    s.qkv_w, s.o_w, s.head_w = (ops.Int8Weight(w(o, i, std)) for o, i, std in (
        ((HQ + 2 * HKV) * 128, HIDDEN, 0.06), (HIDDEN, HQ * 128, 0.05), (VOCAB, HIDDEN, 0.15)))
    s.bias = torch.randn((HQ + 2 * HKV) * 128, generator=g).to(BF16).to(dev)
    s.tok = torch.randint(VOCAB, (n,), generator=g).to(dev)
    s.u = torch.rand(n, generator=g).to(dev)
    s.temp = torch.tensor([0.0 if i == 1 else 0.5 + 0.2 * i for i in range(n)], device=dev)
    s.top_k = torch.tensor([0 if i % 2 else 20 + i for i in range(n)], dtype=torch.int32, device=dev)
    s.top_p = torch.tensor([0.9 if i % 3 else 1.0 for i in range(n)], device=dev)
    s.min_p = torch.tensor([0.02 if i % 4 == 0 else 0.0 for i in range(n)], device=dev)
    return s


def _step(s):
    o, r = s.ops, SimpleNamespace()
    r.tok = s.tok.clone()
    r.x = s.embed[s.tok]
    r.xq, r.xs = o.int8_rows(r.x)
    r.qkv = o.int8_matmul(r.xq, r.xs, s.qkv_w, s.bias)
    q, k, v = prefix._views(vars(s), r.qkv)
    r.attn = o.prefix_attention(q, k, v, s.kc, s.vc, s.pt, s.plens, s.bt, s.lens, s.pos, s.cs, s.scale, cu_groups=s.cg,
                                cu_seqlens=s.cu)
    r.aq, r.as_ = o.int8_rows(r.attn)
    r.o = o.int8_matmul(r.aq, r.as_, s.o_w)
    r.h = r.x + r.o
    r.hq, r.hs = o.int8_rows(r.h)
    r.logits = o.int8_matmul(r.hq, r.hs, s.head_w)
    o.sample_tokens(r.logits, s.u, s.temp, s.top_k, s.top_p, s.min_p, out=s.tok)
    s.lens.add_(s.new_dev)
    s.pos.add_(s.step_of)
    return r


def _before(s):
    return dict(kc=s.kc.cpu(), vc=s.vc.cpu(), lens=s.lens.cpu(), pos=s.pos.cpu(), **{
        k: getattr(s, k).cpu() for k in ("pt", "bt", "plens", "cg", "cu", "cs")}, hq=HQ, hkv=HKV, scale=s.scale)


def _check(s, r, before):
    assert torch.equal(r.x.cpu(), s.embed.cpu()[r.tok.cpu()])
    for x, q, sc, w, bias, y in ((r.x, r.xq, r.xs, s.qkv_w, s.bias, r.qkv), (r.attn, r.aq, r.as_, s.o_w, None, r.o),
                                 (r.h, r.hq, r.hs, s.head_w, None, r.logits)):
        wq, ws = int8.codes(x.cpu())
        assert torch.equal(q.cpu().double(), wq)
        assert bool(((sc.cpu().double() - ws).abs() <= 2.0 ** -24 * ws).all())
        int8.check(y, q.cpu().double(), sc.cpu().double(), int8.unpacked(w), w.scale.cpu().double(),
                   None if bias is None else bias.cpu())
    c = dict(before, qkv=r.qkv.cpu())
    want, w, kc, vc = prefix._want(c)
    off = (r.attn.cpu().double() - want).abs()
    assert bool((off <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * w + 1e-30).all())  # (as its own tests derive)
    assert torch.equal(s.vc.cpu(), vc) and bool(((s.kc.cpu().double() - kc.double()).abs() <= 2.0 ** -7 * kc.double().abs() + 1e-30).all())
    x = r.logits.cpu().double().numpy()
    f = lambda t, i: t[i].double().item()  # noqa: E731
    assert s.tok.tolist() == [want_token(x[i], f(s.u, i), f(s.temp, i), int(s.top_k[i]), f(s.top_p, i), f(s.min_p, i))
                              for i in range(s.n)]


@pytest.mark.parametrize("drafts", [0, 1])
def test_step_eager_and_replayed(dev, drafts):
    told = []
    for captured in (False, True):
        s = _state(dev, drafts)
        s.new_dev = s.new.to(dev)
        g = torch.Generator().manual_seed(72)
        graph, tokens = None, []
        for i in range(5):
            s.u.copy_(torch.rand(s.n, generator=g))
            before = _before(s)
            if captured and i:
                if graph is None:
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        r = _step(s)
                graph.replay()
            else:
                r = _step(s)
            torch.cuda.synchronize()
            _check(s, r, before)
            tokens.append((s.tok.tolist(), r.logits.cpu()))
        told.append(tokens)
    for (a, x), (b, y) in zip(*told):
        assert a == b and torch.equal(x, y)
