"""Rotary positions with several axes (pasa_rope_axes): the positions of image and video tokens, without a table."""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import NamedTuple, Optional, Sequence, Union

import torch

from . import _lib
from ._launch import check_cuda, launch, overlaps_itself, wants_grad, written

_DTYPES = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_POS_TYPES = {torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64, torch.float32: _lib.POS_F32,
              torch.float64: _lib.POS_F64}
_PAIRS = {"interleaved": _lib.PAIRS_INTERLEAVED, "halves": _lib.PAIRS_HALVES}


class _Plan(NamedTuple):
    """What a call's arguments other than its tensors come to, checked once for each set of them."""
    axes: tuple
    turned: int            # dimensions
    points: Optional[int]  # of the grid
    where: tuple           # C arguments of the grid
    tail: tuple            # C arguments behind the positions, without the direction


@functools.lru_cache(maxsize=256)
def _plan(axes, theta, pairs, grid, origin) -> _Plan:
    theta = theta if isinstance(theta, tuple) else (theta,) * len(axes)
    if not 1 <= len(axes) <= 4 or any(d < 0 or d % 2 for d in axes) or not 2 <= sum(axes) <= 256:
        raise ValueError(f"axes are 1 to 4 even numbers of dimensions, 2 to 256 together, got {axes}")
    if len(theta) != len(axes) or any(not 0 < t < math.inf for t in theta):
        raise ValueError("theta is one positive number, or one for each axis")
    if pairs not in _PAIRS:
        raise ValueError("pairs is 'interleaved' or 'halves'")
    freqs = [t ** (-2 * i / d) for d, t in zip(axes, theta) for i in range(d // 2)]
    where = points = None
    if grid is not None:
        origin = (0,) * len(axes) if origin is None else origin
        if len(grid) != len(axes) or len(origin) != len(axes) or min(grid) < 0:
            raise ValueError(f"grid {grid} and origin {origin} need one number for each of {len(axes)} axes")
        points = math.prod(grid)
        where = (None, 0, 0, (ctypes.c_int64 * len(grid))(*grid), (ctypes.c_int64 * len(grid))(*origin))
    elif origin is not None:
        raise ValueError("origin goes with grid")
    tail = (len(axes), (ctypes.c_int * len(axes))(*axes), (ctypes.c_double * len(freqs))(*freqs), _PAIRS[pairs])
    return _Plan(axes, sum(axes), points, where, tail)


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


# pasa_rope_tensor, once or twice
_TENSORS = {n: struct.Struct("=" + n * "QQ7q") for n in (1, 2)}


def _apply(tensors, outs, positions, plan, inverse):
    first = tensors[0]
    batch, _, tokens, dim = first.shape
    fields = []
    for x, out in zip(tensors, outs):
        xs, os = x.stride(), out.stride()
        fields += (x.data_ptr(), out.data_ptr(), x.shape[1], xs[0], xs[1], xs[2], os[0], os[1], os[2])
    if positions is None:
        where = plan.where
    else:
        where = (positions.data_ptr(), _POS_TYPES[positions.dtype],
                 positions.stride(0) if positions.dim() == 3 and batch > 1 else 0, None, None)
    launch("pasa_rope_axes", first.device, _TENSORS[len(tensors)].pack(*fields), len(tensors), _DTYPES[first.dtype],
           batch, tokens, dim, *where, *plan.tail, inverse)
    return outs


class _RopeAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, inverse, positions, *tensors):
        ctx.plan, ctx.inverse = plan, inverse
        ctx.save_for_backward(positions)
        return _new(tensors, positions, plan, inverse)

    @staticmethod
    def backward(ctx, *grads):
        given = [g for g in grads if g is not None]
        # a rotation's transpose is its inverse
        turned = iter(_turn(given, ctx.saved_tensors[0], ctx.plan, not ctx.inverse) if given else ())
        return (None, None, None, *(None if g is None else next(turned) for g in grads))


def _new(tensors, positions, plan, inverse):
    rows = [_rows(t) for t in tensors]
    return tuple(_apply(rows, [torch.empty_like(t) for t in rows], positions, plan, inverse))


def _turn(tensors, positions, plan, inverse):
    if wants_grad("rope_axes", *tensors):
        return _RopeAxes.apply(plan, inverse, positions, *tensors)
    return _new(tensors, positions, plan, inverse)


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
    without k), or q and k themselves with ``inplace`` (they must not overlap).  Differentiable in q and k (in
    reverse mode), except under stream capture.
    """
    check_cuda("q", q, 4, _DTYPES)
    tensors = (q,)
    batch, _, tokens, dim = q.shape
    if k is not None:
        check_cuda("k", k, 4, _DTYPES, q.device)
        if k.dtype != q.dtype or (k.shape[0], k.shape[2], k.shape[3]) != (batch, tokens, dim):
            raise ValueError(f"q and k may differ in heads only, got {q.dtype} {tuple(q.shape)} and {k.dtype} "
                             f"{tuple(k.shape)}")
        tensors = (q, k)
    if (positions is None) == (grid is None):
        raise ValueError("give either positions or grid")
    # (numbers, not objects that hold them: plans are found again by their values)
    plan = _plan(tuple(map(int, axes)), tuple(map(float, theta)) if isinstance(theta, (tuple, list)) else float(theta),
                 pairs, None if grid is None else tuple(map(int, grid)),
                 None if origin is None else tuple(map(int, origin)))
    if plan.turned > dim:
        raise ValueError(f"axes {plan.axes} take more than the {dim} dimensions of a head")
    if grid is not None and plan.points != tokens:
        raise ValueError(f"grid {tuple(grid)} has {plan.points} points for {tokens} tokens")
    if positions is not None:
        check_cuda("positions", positions, None, _POS_TYPES, q.device)
        if tuple(positions.shape) not in ((tokens, len(plan.axes)), (batch, tokens, len(plan.axes))):
            raise ValueError(f"positions must be [{tokens}, {len(plan.axes)}] or [{batch}, {tokens}, "
                             f"{len(plan.axes)}], got {tuple(positions.shape)}")
        positions = positions.contiguous()
    inverse = bool(inverse)
    if inplace:
        if wants_grad("rope_axes", *tensors):
            raise ValueError("inplace is not differentiable")
        for name, t in zip("qk", tensors):
            if (dim > 1 and t.stride(3) != 1) or overlaps_itself(t):
                raise ValueError(f"{name} must have unit stride in its last dimension and no broadcast one to be "
                                 "turned in place")
        if k is not None and k.data_ptr() == q.data_ptr() and q.numel():
            raise ValueError("q and k are the same memory: it would be turned twice")
        _apply(tensors, tensors, positions, plan, inverse)
        written(*tensors)
    else:
        tensors = _turn(tensors, positions, plan, inverse)
    return tensors[0] if k is None else tensors
