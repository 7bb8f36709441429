"""GPU test of a worker whose cache is held in 4 bits: WorkerEngine over a
PagedKVCache4 in a worker process, prefill chunks and decode tokens of a lone
slot (q, k, v read in place in the fused rows, the result written into the
slot's staged input buffer), every attention call compared with the definition
in 64 bits on the CPU."""

import math
import threading

import pytest
import torch
import torch.multiprocessing as mp

pytestmark = pytest.mark.gpu


def _worker(shm_name, claim, worker_id, prompt, n_new, gpu_ordered, out, calls):
    """_worker_proc with the cache replaced and its attention calls checked."""
    from swarmlora_amd.worker import batched_ops, paged_attention
    from tests import _kv4
    from tests.test_runtime_gpu import _worker_proc
    paged_attention.PagedKVCache = paged_attention.PagedKVCache4
    plain = batched_ops.WorkerBatchedOps.batch_flash_attention
    seen = {"calls": 0, "staged": 0, "lens": []}

    def checked(slot_ids, qkv, kv, cs, layer, hq, hkv, d, meta, out=None):
        (sid,) = slot_ids
        assert type(kv) is paged_attention.PagedKVCache4
        q, k, v = (t.reshape(-1, h, d).cpu() for t, h in zip(qkv[sid], (hq, hkv, hkv)))
        pages, bt = kv.pages[layer].cpu(), meta["block_tables"].cpu()
        ctx, pos, rows = int(meta["cache_seqlens"][0]), meta["positions"].cpu(), cs.cpu()
        got = plain(slot_ids, qkv, kv, cs, layer, hq, hkv, d, meta, out=out)[sid]
        n = q.shape[0]
        kr, qr = _kv4.rotate(k, rows[pos]), _kv4.rotate(q, rows[pos]).to(torch.bfloat16)
        for t in range(n):
            _kv4.store(pages, bt, 0, int(pos[t]), kr[t], v[t].double())
        assert torch.equal(kv.pages[layer].cpu(), pages)
        want, a = _kv4.attend(qr, pages, bt, [ctx], [0, n], 1 / math.sqrt(d))
        # half a step of bf16, and the probabilities' rounding to bf16 (of terms and sum)
        off = (got.cpu().double().view_as(want) - want).abs()
        assert got.shape == (1, n, hq * d) and bool((off <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * a + 1e-30).all())
        if out is not None:
            assert got.data_ptr() == out[sid].data_ptr()
            seen["staged"] += 1
        seen["calls"] += 1
        seen["lens"].append((ctx, n))
        return {sid: got}

    batched_ops.WorkerBatchedOps.batch_flash_attention = staticmethod(checked)
    _worker_proc(shm_name, claim, worker_id, prompt, n_new, False, out, gpu_ordered)
    calls.put(seen)


@pytest.mark.parametrize("gpu_ordered", [False, True])
def test_engine_over_a_cache_of_four_bits(dev, gpu_ordered):
    from swarmlora_amd import ext_aggregator as agg
    from swarmlora_amd import ext_ipc_queue as extq
    from tests._tiny_model import CFG as c, base_weights
    weights = base_weights(c)
    q = extq.create_queue(512, 512)
    extq.init_batch_control(4)
    agg.init_slot_pool(4, 0, c.hidden, c.inter, c.kv_heads, c.head_dim, c.chunk, 2)
    agg.init_aggregator_begin(c.layers, 0)
    for li, w in enumerate(weights["layers"]):
        agg.init_aggregator_layer(li, *(w[n].to(dev) for n in ("q", "k", "v", "o")), torch.empty(0),
                                  w["gate"].to(dev), w["up"].to(dev), w["down"].to(dev), torch.empty(0))
    agg.init_aggregator_finalize()
    agg.init_embed_lm_head_weights(weights["embed"].to(dev), weights["lm_head"].to(dev))
    agg.init_aggregator_queue(q["shm_name"], 512)
    claim = agg.claim_slot(1)
    loop = threading.Thread(target=agg.aggregator_main_loop_slots, args=(4, 15), daemon=True)
    loop.start()
    ctx = mp.get_context("spawn")
    out, calls = ctx.Queue(), ctx.Queue()
    prompt = torch.randint(0, c.vocab, (20,), generator=torch.Generator().manual_seed(3)).tolist()
    proc = ctx.Process(target=_worker, args=(q["shm_name"], claim, 1, prompt, 3, gpu_ordered, out, calls))
    try:
        proc.start()
        _, rec, toks, err = out.get(timeout=90)
        assert err is None, err
        seen = calls.get(timeout=30)
    finally:
        extq.set_quit(1)
        loop.join(timeout=30)
        proc.join(timeout=30)
        if proc.is_alive():
            proc.kill()
        try:
            agg.release_slot(claim["slot_id"], 1)
        except RuntimeError:
            pass
        agg.cleanup_slot_pool()
        extq.close_queue()
    assert not loop.is_alive() and len(toks) == 3
    assert seen["calls"] == len(rec) * c.layers and seen["staged"] == seen["calls"]
    assert seen["lens"][::c.layers] == [(0, 16), (16, 4), (20, 1), (21, 1)]
