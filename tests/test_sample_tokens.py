"""CPU tests: what swl_sample_tokens_bf16 and its front end refuse."""

import pytest
import torch

P = 4096  # a pointer that is never followed: the checks come first


def _lib():
    from swarmlora_amd import _lib
    return _lib


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null"), (dict(u=None), "null"), (dict(t=None), "null"), (dict(out=None), "null"), (dict(ld=99), "stride"),
    (dict(n=-1), "rows"), (dict(n=65536), "rows"), (dict(v=0), "vocabulary"), (dict(v=(1 << 21) + 1, ld=1 << 22), "vocabulary"),
    (dict(ws=None), "workspace"), (dict(ws=P + 8), "workspace"), (dict(wsb=100), "workspace"),
])
def test_refusals(kw, text):
    lib = _lib().load()
    a = dict(x=P, ld=100, n=3, v=100, u=P, t=P, k=P, p=P, m=P, out=P, ws=P, wsb=1 << 30)
    a.update(kw)
    assert lib.swl_sample_tokens_bf16(*[a[n] for n in ("x", "ld", "n", "v", "u", "t", "k", "p", "m", "out", "ws", "wsb")], None)
    assert text in _lib().last_error()


def test_nothing_to_do_and_workspace():
    lib = _lib().load()
    assert lib.swl_sample_tokens_bf16(None, 100, 0, 100, *[None] * 7, 0, None) == 0
    assert lib.swl_sample_tokens_workspace(0, 100) == 0 and lib.swl_sample_tokens_workspace(2, 100) > 0


def test_front_end_needs_gpu_tensors():
    from swarmlora_amd import ops
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.sample_tokens(torch.zeros(2, 10, dtype=torch.bfloat16), torch.zeros(2), torch.ones(2))
