"""The adapters' C entry points on the host: what they refuse before touching the device."""
import ctypes

import pytest
import torch

from pasa_b200 import _lib, ops

P, BAD = 4096, 4104  # aligned and misaligned fake pointers, never dereferenced


def update(*, x=P, ldx=64, y=P, ldy=32, a=P, b=P, m=5, k=64, n=32, rank=8, adapters=1, rows=P, slots=P, requests=1,
           h=P, out=P, ldo=32):
    return _lib.load().pasa_lora_update(None, x, ldx, y, ldy, a, b, None, m, k, n, rank, adapters, rows, slots, requests,
                                        h, out, ldo)


def backward(*, dy=P, lddy=32, x=P, ldx=64, a=P, b=P, m=5, k=64, n=32, rank=8, adapters=1, rows=P, slots=P, requests=1,
             h=P, base=None, ldbase=0, dx=P, lddx=64, da=P, db=P, workspace=P, size=1 << 30):
    return _lib.load().pasa_lora_update_backward(None, dy, lddy, x, ldx, a, b, None, m, k, n, rank, adapters, rows,
                                                 slots, requests, h, 1, base, ldbase, dx, lddx, da, db, workspace, size)


@pytest.mark.parametrize("call", [update, backward])
def test_refusals_come_before_the_device(call):
    for wrong in (dict(k=60), dict(n=36), dict(rank=4), dict(rank=12), dict(rank=136), dict(rank=0), dict(adapters=0),
                  dict(m=-1), dict(requests=-1), dict(ldx=56), dict(ldx=68), dict(k=0), dict(n=0), dict(m=1 << 31)):
        assert call(**wrong) == _lib.ERR_SHAPE, wrong
    for wrong in (dict(x=None), dict(a=None), dict(b=None), dict(rows=None), dict(slots=None), dict(h=None)):
        assert call(**wrong) == _lib.ERR_NULL, wrong
    for wrong in (dict(x=BAD), dict(a=BAD), dict(b=BAD), dict(h=BAD)):
        assert call(**wrong) == _lib.ERR_ALIGN, wrong


def test_refusals_of_each():
    assert update(y=None) == update(out=None) == _lib.ERR_NULL
    assert update(y=BAD) == update(out=BAD) == _lib.ERR_ALIGN
    assert update(ldy=24) == update(ldo=36) == update(ldo=40) == _lib.ERR_SHAPE  # in place: one stride
    assert backward(dy=BAD) == backward(dx=BAD) == backward(da=BAD) == backward(base=BAD, ldbase=64) == _lib.ERR_ALIGN
    assert backward(lddx=56) == backward(lddy=24) == backward(base=P, ldbase=72) == _lib.ERR_SHAPE


def test_nothing_to_do():
    assert update(m=0) == _lib.OK


def test_h_size():
    n = ctypes.c_size_t()
    lib = _lib.load()
    assert lib.pasa_lora_h_size(10, 24, ctypes.byref(n)) == _lib.OK and n.value == 2 * 10 * 32 * 2
    assert lib.pasa_lora_h_size(10, 20, ctypes.byref(n)) == _lib.ERR_SHAPE
    assert lib.pasa_lora_h_size(10, 24, None) == _lib.ERR_NULL


def test_cpu_tensors_are_refused():
    t = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    rows, slots = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.lora_update(t(4, 8), t(4, 8), t(1, 8, 8), t(1, 8, 8), rows, slots)
