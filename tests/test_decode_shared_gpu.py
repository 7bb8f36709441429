"""GPU parity of the batched decode step whose workers share prompts and sample
from given random numbers, against the CPU oracle's decode_step on the same
pages (a worker's context is its prefix's pages, then its own)."""

import pytest
import torch

from oracle import reference_path as ref
from tests._util import randn, rel_err
from tests.test_sample_tokens_gpu import want_token

pytestmark = pytest.mark.gpu

CTX = [0, 3, 17, 40, 100]
PREFIXES = [(48, 3), (160, 1)]  # whole pages: then the oracle's tables are the two after each other
TOL = 1e-2  # normalised max error of the logits (that of the step without prefixes)


def _decoder(dev, **kw):
    from swarmlora_amd.decode import BatchedDecoder, DecodeShape
    from tests._tiny_model import CFG as c, adapter, base_weights
    shape = DecodeShape(layers=c.layers, hidden=c.hidden, heads=c.heads, kv_heads=c.kv_heads, head_dim=c.head_dim,
                        inter=c.inter, vocab=c.vocab, eps=c.eps, theta=c.theta, block_size=c.block, rank=c.rank,
                        scale=c.scale)
    names = {"q": "self_attn.q_proj", "k": "self_attn.k_proj", "v": "self_attn.v_proj", "o": "self_attn.o_proj",
             "gate": "mlp.gate_proj", "up": "mlp.up_proj", "down": "mlp.down_proj"}
    wts = base_weights()
    ads = [None if w == 2 else {li: {p: m[names[p]] for p in names} for li, m in adapter(w).items()} for w in range(5)]
    pages = {}

    def kv_fill(li, kc, vc, bt):
        assert bt.shape[0] == len(CTX) + len(kw.get("prefixes") or [])
        pages[li] = randn(tuple(kc.shape), 500 + li), randn(tuple(vc.shape), 600 + li)
        kc.copy_(pages[li][0])
        vc.copy_(pages[li][1])

    dec = BatchedDecoder(shape, wts, ads, CTX, [5, 77, 300, 639, 0], dev, max_new=8, kv_fill=kv_fill, **kw)
    return dec, shape, wts, ads, [[pages[li][j].clone() for li in range(c.layers)] for j in range(2)]


def test_shared_prompts_and_sampling(dev):
    g = torch.Generator().manual_seed(9)
    asked = dict(u=torch.zeros(5, device=dev), temperature=torch.tensor([0.0, 0.7, 1.0, 1.3, 0.5], device=dev),
                 top_k=torch.tensor([0, 20, 0, 100, 0], dtype=torch.int32, device=dev),
                 top_p=torch.tensor([1.0, 0.9, 0.95, 1.0, 1.0], device=dev))
    dec, shape, wts, ads, (kc, vc) = _decoder(dev, prefixes=PREFIXES, sampling=asked)
    try:
        cs = ref.cos_sin_cache(ref.rope_inv_freq(shape.head_dim, shape.theta), dec.cos_sin.shape[0])
        of = [0, 0, 0, 1, None]
        before = [48, 48, 48, 160, 0]
        own, pre = dec.block_tables.cpu(), dec.prefix_tables.cpu()
        width = own.shape[1] + 10
        bt = torch.zeros(5, width, dtype=torch.int32)
        for w in range(5):
            row = torch.cat([pre[of[w], :before[w] // 16], own[w]]) if of[w] is not None else own[w]
            bt[w, :len(row)] = row[:width]
        for step in range(5):
            if step == 2:
                dec.capture()
            asked["u"].copy_(torch.rand(5, generator=g))
            ids = dec.ids.reshape(-1).cpu()
            dec.step()
            torch.cuda.synchronize()
            seq = torch.tensor([c + b + step for c, b in zip(CTX, before)], dtype=torch.int32)
            _, lg = ref.decode_step(shape, wts, ads, kc, vc, bt, seq, ids, cs)
            assert rel_err(dec.logits.cpu(), lg) <= TOL, step
            x = dec.logits.cpu().double().numpy()
            a = {k: v.cpu() for k, v in asked.items()}
            assert dec.ids.reshape(-1).tolist() == [
                want_token(x[w], float(a["u"][w]), float(a["temperature"][w]), int(a["top_k"][w]), float(a["top_p"][w]))
                for w in range(5)]
        for li in range(shape.layers):
            assert rel_err(dec.kv.value_caches[li], vc[li]) <= TOL
            assert rel_err(dec.kv.key_caches[li], kc[li]) <= TOL
    finally:
        dec.close()


def test_prefixes_that_end_inside_a_page(dev):
    # 37 and 161 tokens in pages of 16; the oracle has pages of its own, with every
    # worker's tokens one after another
    prefixes, before, of = [(37, 2), (161, 2)], [37, 37, 161, 161, 0], [0, 0, 1, 1, None]
    dec, shape, wts, ads, pages = _decoder(dev, prefixes=prefixes)
    try:
        own, pre = dec.block_tables.cpu(), dec.prefix_tables.cpu()
        width = max((b + c + 8 + 15) // 16 for b, c in zip(before, CTX))
        bt = torch.arange(5 * width, dtype=torch.int32).view(5, width)
        at = lambda row, p: (row[p // 16].long(), p % 16)  # noqa: E731
        held = [[torch.zeros(5 * width, 16, *p.shape[2:], dtype=p.dtype) for p in ps] for ps in pages]
        for w in range(5):
            t = torch.arange(before[w] + CTX[w])
            ctx = t >= before[w]
            for ps, hs in zip(pages, held):
                for p, x in zip(ps, hs):
                    if of[w] is not None:
                        x[at(bt[w], t[~ctx])] = p[at(pre[of[w]], t[~ctx])]
                    x[at(bt[w], t[ctx])] = p[at(own[w], t[ctx] - before[w])]
        cs = ref.cos_sin_cache(ref.rope_inv_freq(shape.head_dim, shape.theta), dec.cos_sin.shape[0])
        for step in range(4):
            if step == 2:
                dec.capture()
            ids = dec.ids.reshape(-1).cpu()
            dec.step()
            torch.cuda.synchronize()
            seq = torch.tensor([c + b + step for c, b in zip(CTX, before)], dtype=torch.int32)
            _, lg = ref.decode_step(shape, wts, ads, *held, bt, seq, ids, cs)
            assert rel_err(dec.logits.cpu(), lg) <= TOL, step
        for li in range(shape.layers):  # the new tokens' keys and values
            for mine, want in ((dec.kv.key_caches[li].cpu(), held[0][li]), (dec.kv.value_caches[li].cpu(), held[1][li])):
                for w in range(5):
                    new = torch.arange(4) + CTX[w]
                    assert rel_err(mine[at(own[w], new)], want[at(bt[w], new + before[w])]) <= TOL
    finally:
        dec.close()


def test_a_prefix_takes_its_pages_once(dev):
    prefixes = [(3000, 3), (161, 1)]
    dec = _decoder(dev, prefixes=prefixes)[0]
    try:
        # 8 tokens to come; pages of 16
        assert dec.kv.num_blocks == sum((c + 8 + 15) // 16 for c in CTX) + 188 + 11
        assert all(t.shape[0] == dec.kv.num_blocks for t in dec.kv.key_caches + dec.kv.value_caches)
        assert dec.block_tables.shape == (5, 7) and dec.prefix_tables.shape == (2, 188)
        assert not dec.kv.free_blocks
        for _ in range(8):
            dec.step()
        torch.cuda.synchronize()
        assert bool(torch.isfinite(dec.logits).all())
    finally:
        dec.close()


@pytest.mark.parametrize("fused", [False, True])
def test_sampling_at_no_temperature_is_the_greedy_step(dev, fused):
    told = []
    for sampling in (None, dict(u=torch.full((5,), 0.7, device=dev), temperature=torch.zeros(5, device=dev))):
        dec = _decoder(dev, fused=fused, sampling=sampling)[0]
        try:
            told.append([dec.step() or dec.ids.reshape(-1).tolist() for _ in range(3)])
        finally:
            dec.close()
    assert told[0] == told[1]


def test_sampling_is_looked_at_when_the_decoder_is_made(dev):
    u, t = torch.zeros(5, device=dev), torch.ones(5, device=dev)
    for kw, error, text in ((dict(u=u), ValueError, "u and temperature"), (dict(temperature=t), ValueError, "u and temperature"),
                            (dict(u=u, temperature=t, topk=t), ValueError, "u and temperature"),
                            (dict(u=u, temperature=t[:4]), ValueError, "temperature must be contiguous"),
                            (dict(u=u, temperature=t, top_k=t), TypeError, "top_k"),
                            (dict(u=u, temperature=t, top_p=t.cpu()), (ValueError, RuntimeError), "top_p"),
                            (dict(u=u, temperature=t, out=t.long()), ValueError, "u and temperature")):
        with pytest.raises(error, match=text):
            _decoder(dev, sampling=kw)


def test_refusals(dev):
    for kw, text in ((dict(prefixes=[(16, 2)], fused=False), "fused"), (dict(prefixes=[(0, 2)]), "at least one"),
                     (dict(prefixes=[(16, 4), (16, 2)]), "at least one")):
        with pytest.raises(ValueError, match=text):
            _decoder(dev, **kw)
