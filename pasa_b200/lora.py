"""Low-rank adapters of many requests beside a shared projection (pasa_lora_update) and their gradients."""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from . import _lib
from ._launch import check_cuda, check_target, launch, refuse_tangents, wants_grad, written

_BF16 = (torch.bfloat16,)
_I32 = (torch.int32,)
_F32 = (torch.float32,)


def _matrix(t: torch.Tensor, name: str, device=None):
    """t [..., C] as rows of one stride that a kernel can read: (2-D tensor, row stride).  Copies what it has to."""
    check_cuda(name, t, None, _BF16, device)
    if t.dim() < 2:
        raise ValueError(f"{name} must be [rows, columns] or [..., columns], got shape {tuple(t.shape)}")
    m = t if t.dim() == 2 else t.reshape(t.shape[:-1].numel(), t.shape[-1])
    rows, cols = m.shape
    step, unit = m.stride()
    if unit == 1 and not m.data_ptr() & 15:
        if rows <= 1:
            return m, cols
        if step >= cols and not step & 7:
            return m, step
    return torch.empty((rows, cols), dtype=m.dtype, device=m.device).copy_(m), cols


def _target(t: torch.Tensor, name: str, shape, device):
    """A tensor that is written in place, as rows of one stride."""
    check_cuda(name, t, None, _BF16, device)
    check_target(name, t)
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    try:
        m = t.view(shape[:-1].numel(), shape[-1])
    except RuntimeError:
        raise ValueError(f"{name} is written in place: its rows must have one stride") from None
    rows, cols = m.shape
    step, unit = m.stride()
    if m.numel() and (unit != 1 or m.data_ptr() & 15 or (rows > 1 and (step < cols or step & 7))):
        raise ValueError(f"{name} is written in place: it must be 16-byte aligned with unit column stride and a row "
                         "stride that is a multiple of 8")
    return m, cols if rows <= 1 else step


def _overlap(a: torch.Tensor, lda: int, b: torch.Tensor, ldb: int) -> bool:
    """Whether two bf16 matrices (rows lda and ldb values apart) share memory.  Columns of the same rows beside one
    another do not; of rows that lie differently among one another that is not found out."""
    if not a.numel() or not b.numel():
        return False
    at = (a.data_ptr() - b.data_ptr()) // 2
    if at >= (b.shape[0] - 1) * ldb + b.shape[1] or -at >= (a.shape[0] - 1) * lda + a.shape[1]:
        return False
    steps = {ld for m, ld in ((a, lda), (b, ldb)) if m.shape[0] > 1}
    if len(steps) != 1:
        return True
    step = steps.pop()
    return at % step < b.shape[1] or at % step + a.shape[1] > step


@functools.lru_cache(maxsize=256)
def _workspace_bytes(m, k, n, rank, adapters, requests, index: int) -> int:
    size = ctypes.c_size_t()
    with torch.cuda.device(index):
        _lib.check("pasa_lora_backward_workspace_size", _lib.load().pasa_lora_backward_workspace_size(
            m, k, n, rank, adapters, requests, ctypes.byref(size)))
    return size.value


class _Call:
    """The checked arguments that the forward and the gradient share."""

    def __init__(self, x, a, b, rows, slots, scale):
        self.x, self.ldx = _matrix(x, "x")
        device = self.device = x.device
        check_cuda("a", a, 3, _BF16, device)
        check_cuda("b", b, 3, _BF16, device)
        check_cuda("rows", rows, 1, _I32, device)
        check_cuda("slots", slots, 1, _I32, device)
        self.m, self.k = self.x.shape
        self.adapters, self.rank, k = a.shape
        self.n = b.shape[1]
        if k != self.k or b.shape[0] != self.adapters or b.shape[2] != self.rank:
            raise ValueError(f"a must be [adapters, rank, {self.k}] and b [adapters, columns, rank], got "
                             f"{tuple(a.shape)} and {tuple(b.shape)}")
        if self.k % 8 or self.n % 8 or self.rank % 8 or not 8 <= self.rank <= 128 or not self.k or not self.n:
            raise ValueError(f"the columns of x and y and the rank must be multiples of 8 and the rank 8 to 128, got "
                             f"{self.k}, {self.n} and {self.rank}")
        if not 1 <= self.adapters <= 4096:
            raise ValueError(f"1 to 4096 adapters, got {self.adapters}")
        self.requests = slots.shape[0]
        if rows.shape[0] != self.requests + 1:
            raise ValueError(f"rows must hold {self.requests + 1} offsets for {self.requests} requests, got "
                             f"{rows.shape[0]}")
        self.scale = None
        if scale is not None:
            check_cuda("scale", scale, 1, _F32, device)
            if scale.shape[0] != self.adapters:
                raise ValueError(f"scale must hold one number for each of {self.adapters} adapters")
            self.scale = scale.contiguous()
        self.a, self.b, self.rows, self.slots = a.contiguous(), b.contiguous(), rows.contiguous(), slots.contiguous()
        if (self.a.data_ptr() | self.b.data_ptr()) & 15:
            raise ValueError("a and b must be 16-byte aligned")

    def h(self):
        return torch.empty((2, self.m, -(-self.rank // 16) * 16), dtype=torch.bfloat16, device=self.device)

    @property
    def weights(self):
        return self.a.data_ptr(), self.b.data_ptr(), None if self.scale is None else self.scale.data_ptr()

    @property
    def sizes(self):
        return (self.m, self.k, self.n, self.rank, self.adapters, self.rows.data_ptr(), self.slots.data_ptr(),
                self.requests)


def _forward(call: _Call, y, out):
    base, ldy = _matrix(y, "y", call.device)
    if base.shape != (call.m, call.n):
        raise ValueError(f"y must have {call.m} rows of {call.n} columns, got shape {tuple(y.shape)}")
    given = out is not None
    if not given:
        out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
        target, ldo = out, call.n
    else:
        target, ldo = _target(out, "out", y.shape, call.device)
        if _overlap(target, ldo, call.x, call.ldx):
            raise ValueError("out is x or overlaps it")
        if (target.data_ptr() != base.data_ptr() or ldo != ldy) and _overlap(target, ldo, base, ldy):
            raise ValueError("out overlaps y: it may be y itself")
    h = call.h()
    launch("pasa_lora_update", call.device, call.x.data_ptr(), call.ldx, base.data_ptr(), ldy, *call.weights,
           *call.sizes, h.data_ptr(), target.data_ptr(), ldo)
    if given:
        written(out)
    return out, h


def _backward(call: _Call, dy, x_shape, h, dx, need_x, need_a, need_b):
    grad, lddy = _matrix(dy, "dy", call.device)
    if grad.shape != (call.m, call.n):
        raise ValueError(f"dy must have {call.m} rows of {call.n} columns, got shape {tuple(dy.shape)}")
    base, ldbase, adds = 0, 0, dx is not None
    if adds:
        target, lddx = _target(dx, "dx", x_shape, call.device)
        if _overlap(target, lddx, call.x, call.ldx) or _overlap(target, lddx, grad, lddy):
            raise ValueError("dx is x or dy, or overlaps one of them")
        base, ldbase = target.data_ptr(), lddx
    elif need_x:
        dx = torch.empty(x_shape, dtype=torch.bfloat16, device=call.device)
        target, lddx = dx, call.k
    given = h is not None
    if given:
        check_cuda("h", h, 3, _BF16, call.device)
        if h.shape != (2, call.m, -(-call.rank // 16) * 16) or not h.is_contiguous():
            raise ValueError("h is not what lora_update returned for these arguments")
    else:
        h = call.h()
    da = torch.empty_like(call.a) if need_a else None
    db = torch.empty_like(call.b) if need_b else None
    size = _workspace_bytes(call.m, call.k, call.n, call.rank, call.adapters, call.requests, call.device.index)
    workspace = torch.empty(size, dtype=torch.uint8, device=call.device)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    launch("pasa_lora_update_backward", call.device, grad.data_ptr(), lddy, call.x.data_ptr(), call.ldx, *call.weights,
           *call.sizes, h.data_ptr(), int(given), base or None, ldbase, target.data_ptr() if dx is not None else None,
           lddx if dx is not None else 0, ptr(da), ptr(db), workspace.data_ptr(), size)
    if adds:
        written(dx)
    return dx, da, db


class _LoraUpdate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, a, b, rows, slots, scale):
        out, h = _forward(_Call(x, a, b, rows, slots, scale), y, None)
        ctx.save_for_backward(x, a, b, rows, slots, scale, h)
        ctx.mark_non_differentiable(h)
        return out, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _):
        x, a, b, rows, slots, scale, h = ctx.saved_tensors
        need_y, need_x, need_a, need_b = ctx.needs_input_grad[:4]
        dx = da = db = None
        if need_x or need_a or need_b:
            dx, da, db = _backward(_Call(x, a, b, rows, slots, scale), dy, x.shape, h, None, need_x, need_a, need_b)
        return dy if need_y else None, dx, da, db, None, None, None


def lora_update(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, rows: torch.Tensor,
                slots: torch.Tensor, scale: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None,
                return_h: bool = False):
    """Adds the requests' low-rank adapters to a shared projection's output y of x:

        out[i] = y[i] + scale[s] * (x[i] A_s^T) B_s^T    for the rows i of a request with adapter s.

    x: [..., K], y: [..., N] bf16 CUDA tensors with the same rows (the leading dimensions, flattened); a: [S, R, K]
    and b: [S, N, R] bf16, the adapters; ``scale``: fp32 [S], or None for 1.  ``rows`` int32 [Q + 1] and ``slots``
    int32 [Q], both on the GPU and read there: request q owns the rows ``rows[q]`` to ``rows[q + 1]`` and the adapter
    ``slots[q]``, or none where that is outside [0, S).  ``rows`` must not decrease.  Rows of no request keep y.
    K, N and R are multiples of 8, R at most 128 (other ranks: pad with zeros), S at most 4096.

    Returns a new tensor like y, or ``out`` (``out=y`` updates in place); with ``return_h`` also the scaled x A^T that
    ``lora_update_backward`` takes.  Sums are fp32 and the result is rounded once.  Differentiable in y, x, a and b
    (in reverse mode), except under stream capture (capture ``lora_update_backward``).
    """
    if torch.is_grad_enabled() and isinstance(scale, torch.Tensor) and scale.requires_grad:
        raise ValueError("lora_update has no gradient for scale")
    refuse_tangents("lora_update", scale)
    if wants_grad("lora_update", y, x, a, b):
        if out is not None:
            raise ValueError("out is not differentiable")
        result, h = _LoraUpdate.apply(y, x, a, b, rows, slots, scale)
    else:
        result, h = _forward(_Call(x, a, b, rows, slots, scale), y, out)
    return (result, h) if return_h else result


def lora_update_backward(dy: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, rows: torch.Tensor,
                         slots: torch.Tensor, scale: Optional[torch.Tensor] = None, *,
                         h: Optional[torch.Tensor] = None, dx: Optional[torch.Tensor] = None):
    """The gradients of ``lora_update`` from dy, the gradient of its result: (dx, da, db), like x, a and b.

        dx = scale dy B A,    da = scale B^T dy^T x,    db = scale dy^T x A^T

    da and db are summed over all rows of an adapter in a fixed order and are zero for one without rows; dx is zero on
    rows without an adapter.  ``dx``: a tensor like x that the gradient is added to in place (the projection's own);
    without it a new one.  ``h``: the second result of ``lora_update(..., return_h=True)``; without it it is computed
    again.  y's gradient is dy itself.  No autograd: for explicit training steps, captured ones among them.
    """
    refuse_tangents("lora_update_backward", dy, x, a, b, scale, h, dx)
    call = _Call(x, a, b, rows, slots, scale)
    return _backward(call, dy, x.shape, h, dx, True, True, True)
