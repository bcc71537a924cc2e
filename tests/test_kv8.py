"""The 8-bit cache's C entry points on the host: what they refuse before touching the device."""
import ctypes

import pytest
import torch

from pasa_b200 import _lib, ops

P, BAD = 4096, 4104  # aligned and misaligned fake pointers, never dereferenced


def strides(*s):
    return (ctypes.c_int64 * 3)(*s)


GOOD = strides(64, 64, 64)


def write(*, k=P, ks=GOOD, v=P, vs=GOOD, kc=P, vc=P, ksc=P, vsc=P, pages=4, heads=2, dim=64, table=P, width=2, starts=P,
          counts=None, batch=1, tokens=3):
    return _lib.load().pasa_kv8_write(None, k, ks, v, vs, kc, vc, ksc, vsc, pages, heads, dim, table, width, starts,
                                      counts, batch, tokens)


def attend(*, q=P, qs=GOOD, kc=P, vc=P, ksc=P, vsc=P, pages=4, heads=2, dim=64, table=P, width=2, lengths=P, batch=1,
           queries=3, group=2, scale=0.1, out=P, os=GOOD, workspace=P, size=1 << 30):
    return _lib.load().pasa_kv8_attention(None, q, qs, kc, vc, ksc, vsc, pages, heads, dim, table, width, lengths, batch,
                                          queries, group, scale, out, os, workspace, size)


@pytest.mark.parametrize("call", [write, attend])
def test_the_cache(call):
    assert call(dim=96) == _lib.ERR_UNSUPPORTED
    for wrong in (dict(pages=-1), dict(heads=0), dict(heads=1 << 15), dict(width=-1), dict(batch=-1),
                  dict(batch=1 << 16), dict(pages=1 << 31), dict(width=1 << 26)):
        assert call(**wrong) == _lib.ERR_SHAPE, wrong
    for wrong in (dict(kc=None), dict(vc=None), dict(ksc=None), dict(vsc=None), dict(table=None)):
        assert call(**wrong) == _lib.ERR_NULL, wrong
    assert call(kc=BAD) == call(vc=BAD) == _lib.ERR_ALIGN


def test_write():
    assert write(tokens=-1) == _lib.ERR_SHAPE
    assert write(k=None) == write(v=None) == write(ks=None) == write(starts=None) == _lib.ERR_NULL
    assert write(k=BAD) == write(vs=strides(64, 64, 68)) == _lib.ERR_ALIGN
    assert write(tokens=0) == write(batch=0) == _lib.OK


def test_attend():
    for wrong in (dict(queries=-1), dict(group=0), dict(queries=1 << 30), dict(scale=0.0), dict(scale=-1.0),
                  dict(scale=float("nan")), dict(scale=float("inf"))):
        assert attend(**wrong) == _lib.ERR_SHAPE, wrong
    assert attend(q=None) == attend(out=None) == attend(lengths=None) == attend(os=None) == _lib.ERR_NULL
    assert attend(q=BAD) == attend(out=BAD) == attend(qs=strides(4, 64, 64)) == attend(workspace=BAD) == _lib.ERR_ALIGN
    assert attend(workspace=None) == _lib.ERR_WORKSPACE
    assert attend(queries=0) == attend(batch=0) == _lib.OK
    n = ctypes.c_size_t()
    assert _lib.load().pasa_kv8_attention_workspace_size(96, ctypes.byref(n)) == _lib.ERR_UNSUPPORTED
    assert _lib.load().pasa_kv8_attention_workspace_size(64, None) == _lib.ERR_NULL


def test_cpu_tensors_are_refused():
    cache = [torch.zeros(2, 1, 64, 64).to(torch.float8_e4m3fn) for _ in range(2)] + [torch.ones(2, 1) for _ in range(2)]
    table, one = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 1, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv8_write(cache, q, q, table, one)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv8_attention(q, cache, table, one)
