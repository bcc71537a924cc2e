"""Rotary positions with several axes (pasa_rope_axes): the positions of image and video tokens, without a table."""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._launch import check_cuda, launch, overlaps_itself, wants_grad

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_POS_TYPES = {torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64, torch.float32: _lib.POS_F32,
              torch.float64: _lib.POS_F64}
_PAIRS = {"interleaved": _lib.PAIRS_INTERLEAVED, "halves": _lib.PAIRS_HALVES}


@functools.lru_cache(maxsize=64)
def _axes(axes: Tuple[int, ...], theta: Tuple[float, ...]):
    """The axes' dimensions and their pairs' frequencies theta^(-2i/d) as C arrays."""
    if not 1 <= len(axes) <= 4 or any(d < 0 or d % 2 for d in axes) or not 2 <= sum(axes) <= 256:
        raise ValueError(f"axes are 1 to 4 even numbers of dimensions, 2 to 256 together, got {axes}")
    if len(theta) != len(axes) or any(not t > 0 for t in theta):
        raise ValueError("theta is one positive number, or one for each axis")
    freqs = [t ** (-2 * i / d) for d, t in zip(axes, theta) for i in range(d // 2)]
    return (ctypes.c_int * len(axes))(*axes), (ctypes.c_double * len(freqs))(*freqs)


def _check(name, t, like=None):
    check_cuda(name, t, 4, _DTYPES)
    if like is not None:
        if t.device != like.device or t.dtype != like.dtype:
            raise ValueError("q and k must share one dtype and device")
        if (t.shape[0], t.shape[2], t.shape[3]) != (like.shape[0], like.shape[2], like.shape[3]):
            raise ValueError(f"q and k may differ in heads only, got {tuple(like.shape)} and {tuple(t.shape)}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.shape[3] == 1 or t.stride(3) == 1 else t.contiguous()


def _apply(tensors, outs, positions, cfg):
    axes, theta, grid, origin, pairs, inverse = cfg
    c_axes, c_freqs = _axes(axes, theta)
    first = tensors[0]
    batch, _, tokens, dim = first.shape
    args = (_lib.RopeTensor * len(tensors))()
    for a, x, out in zip(args, tensors, outs):
        a.x, a.out, a.heads = x.data_ptr(), out.data_ptr(), x.shape[1]
        a.x_stride[:] = x.stride()[:3]
        a.out_stride[:] = out.stride()[:3]
    if grid is not None:
        where = (None, 0, 0, (ctypes.c_int64 * len(grid))(*grid), (ctypes.c_int64 * len(grid))(*origin))
    else:
        where = (positions.data_ptr(), _POS_TYPES[positions.dtype],
                 positions.stride(0) if positions.dim() == 3 and batch > 1 else 0, None, None)
    launch("pasa_rope_axes", first.device, args, len(tensors), _DTYPES[first.dtype], batch, tokens, dim, *where,
           len(axes), c_axes, c_freqs, pairs, int(inverse))
    return outs


class _RopeAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, positions, *tensors):
        ctx.cfg = cfg
        ctx.save_for_backward(positions)
        return _new(tensors, positions, cfg)

    @staticmethod
    def backward(ctx, *grads):
        cfg = ctx.cfg[:-1] + (not ctx.cfg[-1],)  # a rotation's transpose is its inverse
        given = [g for g in grads if g is not None]
        turned = iter(_turn(given, ctx.saved_tensors[0], cfg) if given else ())
        return (None, None, *(None if g is None else next(turned) for g in grads))


def _new(tensors, positions, cfg):
    rows = [_rows(t) for t in tensors]
    return tuple(_apply(rows, [torch.empty_like(t) for t in rows], positions, cfg))


def _turn(tensors, positions, cfg):
    if wants_grad("rope_axes", *tensors):
        return _RopeAxes.apply(cfg, positions, *tensors)
    return _new(tensors, positions, cfg)


def rope_axes(q: torch.Tensor, k: Optional[torch.Tensor] = None, *, axes: Sequence[int],
              positions: Optional[torch.Tensor] = None, grid: Optional[Sequence[int]] = None,
              origin: Optional[Sequence[int]] = None, theta: Union[float, Sequence[float]] = 10000.0,
              pairs: str = "interleaved", inverse: bool = False, inplace: bool = False):
    """Turns the pairs of the first ``sum(axes)`` dimensions of q (and k) by their tokens' positions.

    q, k: [B, H, T, D] CUDA tensors, bf16 or fp32, any strides (a token-major [B, T, H, D] tensor is passed as
    ``x.transpose(1, 2)``, a sequence whose text stays unturned as ``x[:, :, :video]``); they may differ in heads.
    ``axes``: even numbers of dimensions of the frame, row, column, ... axis; pair i of an axis of d dimensions has
    the frequency ``theta ** (-2 i / d)`` (``theta``: one number, or one for each axis).  The dimensions behind the
    axes are kept.  ``pairs``: "interleaved" pairs the dimensions (2p, 2p + 1), "halves" (p, p + sum(axes) / 2).

    The positions are either ``positions`` ([T, axes] or [B, T, axes], int32, int64, fp32 or fp64), or those of the
    row-major ``grid`` (one size for each axis, T points) counted from ``origin`` (zeros by default).

    ``inverse`` turns back, which is also the gradient: d(rope)/dx applied to dy is ``rope_axes(dy, inverse=True)``.
    Angles are formed in fp64, the rotation in fp32, and rounded once.  Returns new tensors like q and k (one tensor
    without k), or q and k themselves with ``inplace``.  Differentiable in q and k, except under stream capture.
    """
    _check("q", q)
    tensors = [q]
    if k is not None:
        _check("k", k, q)
        tensors.append(k)
    axes = tuple(int(d) for d in axes)
    theta = tuple(float(t) for t in theta) if isinstance(theta, (tuple, list)) else (float(theta),) * len(axes)
    _axes(axes, theta)
    batch, _, tokens, dim = q.shape
    if sum(axes) > dim:
        raise ValueError(f"axes {axes} take more than the {dim} dimensions of a head")
    if pairs not in _PAIRS:
        raise ValueError("pairs is 'interleaved' or 'halves'")
    if (positions is None) == (grid is None):
        raise ValueError("give either positions or grid")
    if positions is not None:
        if origin is not None:
            raise ValueError("origin goes with grid")
        check_cuda("positions", positions, None, _POS_TYPES, q.device)
        if tuple(positions.shape) not in ((tokens, len(axes)), (batch, tokens, len(axes))):
            raise ValueError(f"positions must be [{tokens}, {len(axes)}] or [{batch}, {tokens}, {len(axes)}], "
                             f"got {tuple(positions.shape)}")
        positions = positions.contiguous()
    else:
        grid = tuple(int(n) for n in grid)
        origin = (0,) * len(axes) if origin is None else tuple(int(n) for n in origin)
        points = 1
        for n in grid:
            points *= n
        if len(grid) != len(axes) or len(origin) != len(axes) or min(grid) < 0 or points != tokens:
            raise ValueError(f"grid {grid} and origin {origin} need one number for each of {len(axes)} axes, and "
                             f"{tokens} points")
    cfg = (axes, theta, grid, origin, _PAIRS[pairs], bool(inverse))
    if inplace:
        if wants_grad("rope_axes", *tensors):
            raise ValueError("inplace is not differentiable")
        for name, t in zip("qk", tensors):
            if (dim > 1 and t.stride(3) != 1) or overlaps_itself(t):
                raise ValueError(f"{name} must have unit stride in its last dimension and no broadcast one to be "
                                 "turned in place")
        if k is not None and k.data_ptr() == q.data_ptr() and q.numel():
            raise ValueError("q and k are the same memory: it would be turned twice")
        _apply(tensors, tensors, positions, cfg)
    else:
        tensors = _turn(tensors, positions, cfg)
    return tensors[0] if k is None else tuple(tensors)
