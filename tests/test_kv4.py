"""CPU tests of the 4-bit KV cache: what its entry points refuse (before any
device call), and the test oracle's own encoding."""

import ctypes
import math

import pytest
import torch

from tests import _kv4


def _lib():
    from swarmlora_amd import _lib
    return _lib


def test_record_size_and_workspace():
    from swarmlora_amd import ops
    lib = _lib().load()
    assert lib.swl_kv4_record_bytes() == ops.KV4_RECORD == _kv4.REC
    assert lib.swl_kv4_attention_workspace(0, 0, 0, 1, 8, 2, 64) == 0
    # a table of at most one part needs none; a long one does, bounded whatever its length
    assert lib.swl_kv4_attention_workspace(4, 4, 0, 1, 32, 8, 16) == 0
    big = lib.swl_kv4_attention_workspace(28, 28, 1, 1, 32, 8, 1 << 20)
    assert 0 < big == lib.swl_kv4_attention_workspace(28, 28, 1, 1, 32, 8, 1 << 24) < 1 << 28


P = 4096  # a pointer that is never followed: the checks come first


def _append(lib, **kw):
    a = dict(q=P, qs=1024, k=P, ks=256, v=P, vs=256, qo=P, nseq=2, ntok=4, cu=None, hq=8, hkv=2, d=128, pages=P, nb=4,
             bs=16, bt=P, mb=2, lens=P, pos=P, cs=P, mp=10)
    a.update(kw)
    return lib.swl_kv4_append_bf16(a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["qo"], a["nseq"], a["ntok"], a["cu"],
                                   a["hq"], a["hkv"], a["d"], a["pages"], a["nb"], a["bs"], a["bt"], a["mb"], a["lens"],
                                   a["pos"], a["cs"], a["mp"], None)


@pytest.mark.parametrize("kw,text", [
    (dict(d=64), "head_dim"), (dict(bs=24), "multiple of 16"), (dict(bs=0), "multiple of 16"), (dict(nb=0), "page geometry"),
    (dict(mb=0), "page geometry"), (dict(hkv=0), "head counts"), (dict(hq=0), "head counts"), (dict(qo=None), "go together"),
    (dict(pos=None), "go together"), (dict(mp=0), "go together"), (dict(k=None), "null"), (dict(pages=None), "null"),
    (dict(lens=None), "null"), (dict(ks=255), "strides"), (dict(qs=1016), "strides"), (dict(vs=260), "aligned"),
    (dict(k=P + 2), "aligned"), (dict(pages=P + 8), "aligned"), (dict(ntok=5), "as many tokens"), (dict(nseq=-1), "count"),
    (dict(cs=P + 4), "aligned"), (dict(mb=1 << 40), "page geometry"), (dict(qs=1280, qo=P), "rows are hq"),
    (dict(ntok=1 << 25), "token count"),
])
def test_append_refusals(kw, text):
    lib = _lib().load()
    assert _append(lib, **kw) != 0
    assert text in _lib().last_error()


def test_nothing_to_do_is_no_error():
    lib = _lib().load()
    assert _append(lib, nseq=0, ntok=0) == 0
    assert _append(lib, ntok=0) == 0


@pytest.mark.parametrize("kw,text", [
    (dict(hq=7), "head counts"), (dict(d=256), "head_dim"), (dict(scale=0.0), "softmax_scale"),
    (dict(scale=-1.0), "softmax_scale"), (dict(scale=math.inf), "softmax_scale"), (dict(scale=math.nan), "softmax_scale"),
    (dict(mq=0), "max_q_len"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(qs=1000), "aligned"),
    (dict(ws=None), "workspace"), (dict(wsb=100), "workspace"), (dict(bs=8), "multiple of 16"), (dict(q=P + 2), "aligned"),
    (dict(out=P), "must not be q"), (dict(nseq=1, ntok=1 << 24, hq=256, hkv=256, qs=1 << 15), "too many rows"),
])
def test_attention_refusals(kw, text):
    lib = _lib().load()
    a = dict(q=P, qs=1024, nseq=2, ntok=4, cu=None, mq=2, hq=8, hkv=2, d=128, pages=P, nb=4, bs=16, bt=P, mb=4096, lens=P,
             scale=0.1, out=2 * P, ws=P, wsb=1 << 40)
    a.update(kw)
    rc = lib.swl_kv4_attention_bf16(a["q"], a["qs"], a["nseq"], a["ntok"], a["cu"], a["mq"], a["hq"], a["hkv"], a["d"],
                                    a["pages"], a["nb"], a["bs"], a["bt"], a["mb"], a["lens"], a["scale"], a["out"], a["ws"],
                                    a["wsb"], None)
    assert rc != 0 and text in _lib().last_error()


def test_read_refusals():
    lib = _lib().load()
    args = lambda **kw: [kw.get(n, v) for n, v in (  # noqa: E731
        ("pages", P), ("nb", 4), ("bs", 16), ("bt", P), ("mb", 2), ("starts", P), ("nseq", 1), ("ntok", 3), ("cu", None),
        ("hkv", 2), ("d", 128), ("k", P), ("v", P), ("st", None))]
    for kw, text in ((dict(d=96), "head_dim"), (dict(k=None), "aligned"), (dict(v=P + 4), "aligned"), (dict(bs=20), "16"),
                     (dict(starts=None), "null")):
        assert lib.swl_kv4_read_bf16(*args(**kw)) != 0 and text in _lib().last_error()


def test_python_front_end_needs_gpu_tensors():
    from swarmlora_amd import ops
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.kv4_pages(4, 24, 2, "cpu")
    pages = ops.kv4_pages(4, 32, 2, "cpu")
    assert pages.shape == (4, 2, 2, 2176) and pages.dtype == torch.uint8
    t = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16)
    bt, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.kv4_append(t, t, pages, bt, lens)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.kv4_attention(t, pages, bt, lens, 0.1)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.kv4_read(pages, bt, lens, 1)


def test_oracle_encoding_is_nearest_and_least():
    """The oracle's codes: every value is at the nearest grid point of the
    least scale that holds the group's largest under 7."""
    x = torch.randn(50, 128, dtype=torch.float64) * torch.logspace(-5, 5, 50, dtype=torch.float64).unsqueeze(1)
    code, b = _kv4.encode(x)
    y = _kv4.decode(code, b)
    s = torch.exp2(b.double() - 127).repeat_interleave(32, -1)
    top = (x / s).abs().unflatten(-1, (4, 32)).amax(-1)
    assert bool(((top >= 3.5) & (top < 7)).all())
    grid = torch.cat([_kv4.MAGS, -_kv4.MAGS])
    best = ((x / s).unsqueeze(-1).clamp(-6, 6) - grid).abs().amin(-1)
    assert torch.allclose(((x / s).clamp(-6, 6) - y / s).abs(), best, atol=1e-12)
    # records: every (token, dim) of keys and values has a place of its own
    seen = set()
    for value in (False, True):
        for t in range(16):
            for d in range(128):
                byte, sh = _kv4.code_at(t, d, value)
                seen.add((byte, sh))
            for g in range(4):
                seen.add((_kv4.scale_at(t, g, value), 0))
                seen.add((_kv4.scale_at(t, g, value), 4))
    assert len(seen) == 2 * _kv4.REC


def test_cache_of_four_bits_allocates_as_the_bf16_one():
    from swarmlora_amd.worker.paged_attention import PagedKVCache, PagedKVCache4
    c4 = PagedKVCache4(2, 2, 128, 16, 3, 100, "cpu")
    c16 = PagedKVCache(2, 2, 128, 16, 3, 100, "cpu", torch.bfloat16)
    assert len(c4.pages) == 2 and c4.pages[0].shape == (21, 2, 1, 2176)
    for c in (c4, c16):
        c.ensure_blocks_for_length(1, 17)
        c.ensure_blocks_for_length(0, 100)
        c.ensure_blocks_for_length(1, 33)
        c.advance_seq_lens([0, 1], 5)
    assert c4.slot_block_tables == c16.slot_block_tables and c4.slot_seq_lens == c16.slot_seq_lens
    assert torch.equal(c4.get_block_table_tensor([1, 0]), c16.get_block_table_tensor([1, 0]))
    with pytest.raises(RuntimeError, match="max_seq_len"):
        c4.ensure_blocks_for_length(0, 113)
    with pytest.raises(ValueError, match="128 dims"):
        PagedKVCache4(1, 2, 64, 16, 1, 64, "cpu")
    with pytest.raises(ValueError, match="128 dims"):
        PagedKVCache4(1, 2, 128, 16, 1, 64, "cpu", torch.float16)
    with pytest.raises(ValueError, match="multiple of 16"):
        PagedKVCache4(1, 2, 128, 24, 1, 64, "cpu")
    with pytest.raises(ValueError, match="outside"):
        c4.read(0, 0, 3, 3)
