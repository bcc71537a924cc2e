"""pasa_rope_axes on the host: what it refuses before touching the device, and calls with nothing to do."""
import ctypes
import struct

import pytest
import torch

from pasa_b200 import _lib, ops


def call(*, x=4096, out=4096, heads=2, n_tensors=1, dtype=_lib.BF16, batch=1, tokens=6, dim=16, positions=4096,
         pos_type=_lib.POS_I32, grid=None, axes=(4, 6), freqs=True, pairing=0, n_axes=None):
    strides = (heads * tokens * dim, tokens * dim, dim)
    t = struct.pack("=QQ7q", x or 0, out or 0, heads, *strides, *strides) * 2
    n = len(axes) if n_axes is None else n_axes
    return _lib.load().pasa_rope_axes(
        None, t, n_tensors, dtype, batch, tokens, dim, positions, pos_type, 0,
        None if grid is None else (ctypes.c_int64 * len(grid))(*grid), None, n, (ctypes.c_int * len(axes))(*axes),
        (ctypes.c_double * 128)(*[1.0] * 128) if freqs else None, pairing, 0)


def test_refusals_come_before_the_device():
    assert call(dtype=7) == _lib.ERR_DTYPE
    assert call(pos_type=4) == _lib.ERR_DTYPE
    assert call(positions=None) == _lib.ERR_NULL
    assert call(freqs=False) == _lib.ERR_NULL
    assert call(x=None) == _lib.ERR_NULL
    assert call(n_tensors=3) == _lib.ERR_SHAPE
    assert call(n_axes=0) == _lib.ERR_SHAPE
    assert call(axes=(2, 2, 2, 2, 2)) == _lib.ERR_SHAPE
    assert call(axes=(3, 5)) == _lib.ERR_SHAPE          # odd
    assert call(axes=(0, 0)) == _lib.ERR_SHAPE          # nothing to turn
    assert call(axes=(10, 8)) == _lib.ERR_SHAPE         # more than the head
    assert call(axes=(200, 100), dim=512) == _lib.ERR_SHAPE
    assert call(tokens=-1) == _lib.ERR_SHAPE
    assert call(positions=None, grid=(2, 4)) == _lib.ERR_SHAPE   # 8 points, 6 tokens
    assert call(positions=None, grid=(-2, -3)) == _lib.ERR_SHAPE
    assert call(pairing=2) == _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("nothing", [{"tokens": 0}, {"batch": 0}, {"heads": 0}])
def test_nothing_to_do(nothing):
    assert call(**nothing) == _lib.OK


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope_axes(torch.zeros(1, 1, 4, 8), axes=[8], grid=[4])
