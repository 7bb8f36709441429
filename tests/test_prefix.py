"""CPU tests: what swl_prefix_attention_bf16 and its front end refuse."""

import math

import pytest
import torch

P = 4096  # a pointer that is never followed: the checks come first


def _lib():
    from swarmlora_amd import _lib
    return _lib


def _call(lib, **kw):
    a = dict(q=P, qs=1024, k=P, ks=256, v=P, vs=256, nseq=2, ntok=4, cu=None, hq=8, hkv=2, d=128, kc=P, vc=P, nb=4, bs=16,
             pt=P, mp=8, pl=P, cg=None, ng=1, bt=P, mb=2, lens=P, pos=P, cs=P, maxp=10, scale=0.1, out=2 * P, ws=P, wsb=1 << 40)
    a.update(kw)
    return lib.swl_prefix_attention_bf16(*[a[n] for n in (
        "q", "qs", "k", "ks", "v", "vs", "nseq", "ntok", "cu", "hq", "hkv", "d", "kc", "vc", "nb", "bs", "pt", "mp", "pl", "cg",
        "ng", "bt", "mb", "lens", "pos", "cs", "maxp", "scale", "out", "ws", "wsb")], None)


@pytest.mark.parametrize("kw,text", [
    (dict(d=64), "head_dim"), (dict(hq=7), "head counts"), (dict(hkv=0), "head counts"), (dict(bs=0), "block_size"),
    (dict(nb=0), "page geometry"), (dict(nb=1 << 27, bs=16), "page geometry"), (dict(mb=0), "page geometry"),
    (dict(mb=1 << 40), "page geometry"), (dict(mp=-1), "page geometry"), (dict(scale=0.0), "softmax_scale"),
    (dict(scale=math.nan), "softmax_scale"), (dict(scale=math.inf), "softmax_scale"), (dict(pos=None), "go together"),
    (dict(maxp=0), "go together"), (dict(k=None), "go together"), (dict(q=None), "null"), (dict(out=None), "null"),
    (dict(kc=None), "null"), (dict(bt=None), "null"), (dict(lens=None), "null"), (dict(pt=None), "null"), (dict(pl=None), "null"),
    (dict(mp=0), "null"), (dict(ng=2), "cu_groups"), (dict(ng=0, cg=P), "cu_groups"), (dict(ng=-1), "count"),
    (dict(nseq=-1), "count"), (dict(ntok=1 << 25), "count"), (dict(nseq=1024, ntok=1024), "1024"), (dict(ntok=5), "as many"),
    (dict(qs=1016), "strides"), (dict(ks=248), "strides"), (dict(vs=260), "aligned"), (dict(q=P + 2), "aligned"),
    (dict(cs=P + 4), "aligned"), (dict(vc=P + 8), "aligned"), (dict(out=P), "must not be q"), (dict(ws=None), "workspace"),
    (dict(wsb=100), "workspace"), (dict(ws=P + 8), "workspace"),
    (dict(nseq=1, ntok=1 << 24, hq=256, hkv=1, qs=1 << 15), "too many rows"),
])
def test_refusals(kw, text):
    lib = _lib().load()
    assert _call(lib, **kw) != 0
    assert text in _lib().last_error()


@pytest.mark.parametrize("kw", [
    dict(ntok=1 << 24), dict(ntok=(1 << 24) + 5, pos=None, cs=None, k=None, v=None), dict(ntok=1 << 23, hq=16, hkv=16, ks=2048, vs=2048),
])
def test_more_workgroups_than_a_launch_has(kw):
    # 2^24 of 256 threads: their threads are counted in 32 bits
    lib = _lib().load()
    assert _call(lib, **{**dict(nseq=1, hq=1, hkv=1, qs=2048, ks=128, vs=128, wsb=1 << 60), **kw}) != 0
    assert "too many rows" in _lib().last_error()


def test_nothing_to_do_and_workspace():
    lib = _lib().load()
    assert _call(lib, nseq=0, ntok=0) == 0
    assert _call(lib, ntok=0) == 0
    w = lib.swl_prefix_attention_workspace
    assert w(0, 0, 1, 8, 2, 64, 64, 0) == 0 and w(4, 4, 1, 7, 2, 64, 64, 0) == 0
    # records of tables of any width are bounded
    assert 0 < w(28, 28, 1, 32, 8, 1 << 20, 1 << 20, 0) == w(28, 28, 1, 32, 8, 1 << 24, 1 << 24, 0) < 1 << 28
    assert w(28, 28, 1, 32, 8, 64, 64, 1) - w(28, 28, 1, 32, 8, 64, 64, 0) == 28 * 32 * 256


def test_front_end_needs_gpu_tensors():
    from swarmlora_amd import ops
    t = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16)
    c = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    bt, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.prefix_attention(t, t, t, c, c, bt, n, bt, n, None, None, 0.1)
