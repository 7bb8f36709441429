"""CPU tests: what swl_verify_drafts_bf16 and its front end refuse."""

import pytest
import torch

P = 4096  # a pointer that is never followed: the checks come first


def _lib():
    from swarmlora_amd import _lib
    return _lib


@pytest.mark.parametrize("kw,text", [
    (dict(tgt=None), "null"), (dict(ids=None), "null"), (dict(u=None), "null"), (dict(ul=None), "null"),
    (dict(temp=None), "null"), (dict(tok=None), "null"), (dict(acc=None), "null"), (dict(vocab=0), "vocabulary"),
    (dict(vocab=1 << 31), "vocabulary"), (dict(ldt=99), "strides"), (dict(ldd=99), "strides"), (dict(ws=None), "workspace"),
    (dict(wsb=10), "workspace"), (dict(ws=P + 4), "workspace"), (dict(nd=5), "as many drafts"), (dict(nseq=-1), "count"),
    (dict(md=-1), "count"), (dict(nd=40000), "65535"),
])
def test_refusals(kw, text):
    lib = _lib().load()
    a = dict(tgt=P, ldt=100, drf=P, ldd=100, vocab=100, ids=P, cu=None, nseq=2, nd=4, md=2, temp=P, u=P, ul=P, tok=P, acc=P,
             ws=P, wsb=1 << 30)
    a.update(kw)
    rc = lib.swl_verify_drafts_bf16(*[a[k] for k in ("tgt", "ldt", "drf", "ldd", "vocab", "ids", "cu", "nseq", "nd", "md", "temp",
                                                     "u", "ul", "tok", "acc", "ws", "wsb")], None)
    assert rc != 0 and text in _lib().last_error()


def test_nothing_to_do_and_workspace():
    lib = _lib().load()
    assert lib.swl_verify_drafts_bf16(None, 0, None, 0, 100, None, None, 0, 0, 0, None, None, None, None, None, None, 0,
                                      None) == 0
    assert lib.swl_verify_drafts_workspace(0, 0, 100, 0) == 0
    assert lib.swl_verify_drafts_workspace(4, 8, 100, 1) > lib.swl_verify_drafts_workspace(4, 8, 100, 0) > 0


def test_front_end_needs_gpu_tensors():
    from swarmlora_amd import ops
    z = torch.zeros
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.verify_drafts(z(2, 3, 10, dtype=torch.bfloat16), z(2, 2, dtype=torch.int64), z(2, 2), z(2), z(2))
