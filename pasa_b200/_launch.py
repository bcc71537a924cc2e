"""What the operators with modules of their own share: argument checks, the launch on the tensors' device and its
current stream, and the rule for gradients under stream capture."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib


def check_cuda(name: str, t: torch.Tensor, dims: Optional[int] = None, dtypes=None,
               device: Optional[torch.device] = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (pasa_b200 has no CPU path)")
    if dims is not None and t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(t.shape)}")
    if dtypes is not None and t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)}, got {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")


def launch(fn: str, device: torch.device, *args) -> None:
    """Calls a C entry point on ``device``'s current stream and maps its status to an exception."""
    entry = getattr(_lib.load(), fn)
    index = device.index
    if index == torch._C._cuda_getDevice():
        code = entry(torch._C._cuda_getCurrentRawStream(index), *args)
    else:
        with torch.cuda.device(index):
            code = entry(torch._C._cuda_getCurrentRawStream(index), *args)
    if code:
        _lib.check(fn, code)


def check_operator_errors(device=None) -> None:
    """Raise if a kernel of ``lora_update``, its gradient or the ``kv8`` operators reported an error on ``device``
    since the last call: a wait that it gave up, or a block table or scale that cannot be (synchronises the current
    stream)."""
    index = torch.cuda.current_device() if device is None else torch.device(device).index
    flags = ctypes.c_uint32(0)
    with torch.cuda.device(index):
        _lib.check("pasa_operator_errors", _lib.load().pasa_operator_errors(
            torch.cuda.current_stream().cuda_stream, ctypes.byref(flags)))
    reasons = [text for bit, text in ((_lib.DEVERR_WAIT_TIMEOUT, "a device-side barrier wait timed out"),
                                      (_lib.DEVERR_BAD_PAGE, "a block table names a page that does not exist"),
                                      (_lib.DEVERR_BAD_SCALE, "a page's scale is not a power of two"))
               if flags.value & bit]
    if reasons:
        raise RuntimeError(f"pasa_b200: {', '.join(reasons)} (error word {flags.value:#x})")


def refuse_tangents(fn: str, *tensors) -> None:
    """A tensor with a forward-mode tangent is refused: the kernels would return a result without one."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{fn} has no forward-mode derivative")


def wants_grad(fn: str, *tensors) -> bool:
    """Whether autograd has to see this call.  Forward-mode tangents are refused.  While a stream is captured that is refused: the engine may run leaves'
    accumulation on the stream of an eager graph of the same leaves, which a capture cannot contain."""
    refuse_tangents(fn, *tensors)
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            break
    else:
        return False
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{fn}: autograd is not recorded into a CUDA graph; capture the explicit forward and "
                           "gradient calls under torch.no_grad()")
    return True


def check_target(name: str, t: torch.Tensor) -> None:
    """A tensor that is written in place has no history that autograd would have to know of."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} is written in place and must not require a gradient")


def written(*tensors: torch.Tensor) -> None:
    """Tells autograd that they were written in place: what an operation before has saved of them is no longer valid."""
    torch.autograd.graph.increment_version(tensors)


def overlaps_itself(t: torch.Tensor) -> bool:
    """Whether two elements share memory, for the strides that views have (a broadcast dimension)."""
    return any(size > 1 and stride == 0 for size, stride in zip(t.shape, t.stride()))
