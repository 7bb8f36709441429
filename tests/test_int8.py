"""CPU tests: what the entry points of products in 8-bit integers refuse."""

import pytest
import torch

P = 4096  # a pointer that is never followed: the checks come first


def _lib():
    from swarmlora_amd import _lib
    return _lib


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null"), (dict(q=None), "null"), (dict(s=None), "null"), (dict(ldx=99), "strides"), (dict(ldq=96), "strides"),
    (dict(ldq=120), "aligned"), (dict(q=P + 8), "aligned"), (dict(m=-1), "row count"), (dict(k=0), "131072"),
    (dict(k=(1 << 17) + 1), "131072"),
])
def test_rows_refusals(kw, text):
    lib = _lib().load()
    a = dict(x=P, ldx=100, m=3, k=100, q=P, ldq=112, s=P)
    a.update(kw)
    assert lib.swl_int8_rows_bf16(*[a[n] for n in ("x", "ldx", "m", "k", "q", "ldq", "s")], None)
    assert text in _lib().last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(w=None), "null"), (dict(d=None), "null"), (dict(s=None), "null"), (dict(ld=99), "stride"), (dict(d=P + 8), "aligned"),
    (dict(n=0), "channel count"), (dict(k=(1 << 17) + 1), "131072"),
])
def test_pack_refusals(kw, text):
    lib = _lib().load()
    a = dict(w=P, ld=100, n=3, k=100, d=P, s=P)
    a.update(kw)
    assert lib.swl_int8_pack_bf16(*[a[n] for n in ("w", "ld", "n", "k", "d", "s")], None)
    assert text in _lib().last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), "null"), (dict(qs=None), "null"), (dict(w=None), "null"), (dict(ws=None), "null"), (dict(y=None), "null"),
    (dict(ldq=96), "strides"), (dict(ldy=499), "strides"), (dict(ldq=8200), "aligned"), (dict(q=P + 8), "aligned"),
    (dict(w=P + 8), "aligned"), (dict(y=P + 4), "aligned"), (dict(m=-1), "sizes"), (dict(n=0), "sizes"), (dict(k=1 << 18), "k over"),
    (dict(work=None), "workspace"), (dict(wb=10), "workspace"), (dict(work=P + 8), "workspace"),
])
def test_matmul_refusals(kw, text):
    lib = _lib().load()
    a = dict(q=P, ldq=8192, qs=P, m=200, w=P, ws=P, n=500, k=8192, bias=None, y=P, ldy=500, work=P, wb=1 << 40)
    a.update(kw)
    assert lib.swl_int8_matmul_bf16(*[a[n] for n in ("q", "ldq", "qs", "m", "w", "ws", "n", "k", "bias", "y", "ldy", "work", "wb")],
                                    None)
    assert text in _lib().last_error()


def test_more_workgroups_than_a_launch_has():
    # 2^22 of 1024 threads for a weight, 2^24 of 256 for a product: their threads are
    # counted in 32 bits
    lib = _lib().load()
    assert lib.swl_int8_pack_bf16(P, 1, 1 << 26, 1, P, P, None) and "channel count" in _lib().last_error()
    assert lib.swl_int8_matmul_bf16(P, 16, P, 1, P, P, 1 << 26, 1, None, P, 1 << 26, None, 0, None)
    assert "sizes" in _lib().last_error()
    assert lib.swl_int8_matmul_bf16(P, 16, P, 1 << 30, P, P, 1 << 20, 1, None, P, 1 << 20, None, 0, None)
    assert "too many rows" in _lib().last_error()


def test_nothing_to_do_and_sizes():
    lib = _lib().load()
    assert lib.swl_int8_rows_bf16(None, 100, 0, 100, None, 112, None, None) == 0
    assert lib.swl_int8_matmul_bf16(None, 112, None, 0, None, None, 500, 100, None, None, 500, None, 0, None) == 0
    assert lib.swl_int8_weight_bytes(17, 129) == 2 * 2 * 2048 and lib.swl_int8_weight_bytes(16, 128) == 2048
    assert lib.swl_int8_weight_bytes(0, 1) == 0 and lib.swl_int8_matmul_workspace(0, 5, 5) == 0
    assert lib.swl_int8_matmul_workspace(28, 28672, 4096) == 0


def test_front_end_needs_gpu_tensors():
    from swarmlora_amd import ops
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.int8_rows(torch.zeros(2, 32, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        ops.Int8Weight(torch.zeros(2, 32, dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="Int8Weight"):
        ops.int8_matmul(torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2), torch.zeros(2, 32))
