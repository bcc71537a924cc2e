"""Keys and values in 8 bits, in pages of 64 tokens, and attention over them (pasa_kv8_write, pasa_kv8_attention)."""
from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib
from ._launch import check_cuda, check_target, launch, overlaps_itself, refuse_tangents, written

PAGE = 64
_BF16 = (torch.bfloat16,)
_E4M3 = (torch.float8_e4m3fn,)
_F32 = (torch.float32,)
_I32 = (torch.int32,)


class KV8Cache(NamedTuple):
    """Pages of keys and values [pages, heads, 64, D] in e4m3, and their scales [pages, heads]."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def kv8_cache(pages: int, heads: int, dim: int, device=None) -> KV8Cache:
    """An empty cache of ``pages`` pages of 64 tokens for ``heads`` key/value heads of ``dim`` (64 or 128) dimensions.
    Its pages are handed out by the caller, through the block tables of ``kv8_write`` and ``kv8_attention``."""
    if dim not in (64, 128) or heads < 1 or pages < 0:
        raise ValueError(f"a cache has heads of 64 or 128 dimensions, got {pages} pages of {heads} heads of {dim}")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    k, v = (torch.zeros((pages, heads, PAGE, dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
            for _ in range(2))
    k_scale, v_scale = (torch.ones((pages, heads), dtype=torch.float32, device=device) for _ in range(2))
    return KV8Cache(k, v, k_scale, v_scale)


def _check_cache(cache: Sequence[torch.Tensor], table: torch.Tensor):
    """(C arguments from the cache, sizes, C arguments of the table)"""
    k, v, k_scale, v_scale = cache
    check_cuda("the cache's k", k, 4, _E4M3)
    device = k.device
    check_cuda("the cache's v", v, 4, _E4M3, device)
    check_cuda("the cache's k_scale", k_scale, 2, _F32, device)
    check_cuda("the cache's v_scale", v_scale, 2, _F32, device)
    check_cuda("table", table, 2, _I32, device)
    pages, heads, page, dim = k.shape
    if page != PAGE or dim not in (64, 128) or heads < 1:
        raise ValueError(f"the cache's pages must be [heads, 64, 64 or 128], got {tuple(k.shape[1:])}")
    if v.shape != k.shape or k_scale.shape != (pages, heads) or v_scale.shape != (pages, heads):
        raise ValueError("the cache's k, v and scales do not have the same pages and heads")
    if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
        raise ValueError("the cache must be contiguous")
    return (k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, heads, dim), k


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t itself if its rows can be read with 16-byte loads, else a copy."""
    b, h, s, unit = t.stride()
    if (b | h | s) & 7 or unit != 1 or t.data_ptr() & 15:
        return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
    return t


def _strides(t: torch.Tensor):
    return (ctypes.c_int64 * 3)(*t.stride()[:3])


def _no_grad(fn: str, *tensors: torch.Tensor) -> None:
    refuse_tangents(fn, *tensors)
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f"{fn} has no gradient; call it under torch.no_grad() or on detached tensors")


def kv8_write(cache: Sequence[torch.Tensor], k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
              starts: torch.Tensor, counts: Optional[torch.Tensor] = None) -> None:
    """Rounds new tokens' keys and values into the pages behind the tokens that each request has.

    ``cache``: a ``KV8Cache`` or its four tensors.  k, v: bf16 [B, H, L, D] (any strides).  ``table`` int32 [B, W]:
    token i of request b is row i % 64 of page ``table[b, i // 64]``.  ``starts`` int32 [B]: tokens that request b
    has; ``counts`` int32 [B]: how many of its L new tokens are written (all by default).  All on the GPU, read there.

    A page has one scale for each head, the smallest power of two (2^-100 at least) that brings its tokens to 448 or
    below.  Where a page has earlier tokens its scale does not become smaller and they are rounded again to it.  A
    page that gets an infinity or NaN reads as NaN.  Rows behind the last token keep what they hold.  Two requests
    must not write one page at once.  A needed table entry that is no page is reported by ``check_operator_errors``.
    """
    args, store = _check_cache(cache, table)
    device = store.device
    pages, heads, dim = args[4:]
    check_cuda("k", k, 4, _BF16, device)
    check_cuda("v", v, 4, _BF16, device)
    batch, tokens = k.shape[0], k.shape[2]
    if k.shape != (batch, heads, tokens, dim) or v.shape != k.shape:
        raise ValueError(f"k and v must be [batch, {heads}, tokens, {dim}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if table.shape[0] != batch:
        raise ValueError(f"table must have {batch} rows, got {table.shape[0]}")
    check_cuda("starts", starts, 1, _I32, device)
    if counts is not None:
        check_cuda("counts", counts, 1, _I32, device)
        counts = counts.contiguous()
    if starts.shape[0] != batch or (counts is not None and counts.shape[0] != batch):
        raise ValueError(f"starts and counts must have {batch} entries")
    _no_grad("kv8_write", k, v)
    k, v, table, starts = _rows(k), _rows(v), table.contiguous(), starts.contiguous()
    launch("pasa_kv8_write", device, k.data_ptr(), _strides(k), v.data_ptr(), _strides(v), *args, table.data_ptr(),
           table.shape[1], starts.data_ptr(), None if counts is None else counts.data_ptr(), batch, tokens)
    written(*cache)


@functools.lru_cache(maxsize=None)
def _workspace_bytes(dim: int, index: int) -> int:
    n = ctypes.c_size_t()
    with torch.cuda.device(index):
        _lib.check("pasa_kv8_attention_workspace_size",
                   _lib.load().pasa_kv8_attention_workspace_size(dim, ctypes.byref(n)))
    return n.value


def kv8_attention(q: torch.Tensor, cache: Sequence[torch.Tensor], table: torch.Tensor, lengths: torch.Tensor,
                  scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(q k^T scale) v over the first ``lengths[b]`` tokens of request b's pages; zero where that is 0.

    q: bf16 [B, Hq, L, D] (any strides), Hq a multiple of the cache's heads H: query head h reads head h * H // Hq.
    ``table`` int32 [B, W] as for ``kv8_write``, ``lengths`` int32 [B] (cut at 64 W), both on the GPU and read there.
    ``scale`` is positive, D**-0.5 by default.  Returns a new tensor with q's strides, or ``out`` (its last stride 1,
    the others multiples of 8; it may be q, and must not overlap it otherwise).  Queries enter the products to 8 significant bits (or 2^-17 of the row's largest
    element), probabilities to 11 (or 2^-36 of the largest), sums are fp32.  Has no gradient.
    A needed table entry that is no page, or a scale that is no power of two, makes the rows that need it NaN and is
    reported by ``check_operator_errors``.
    """
    args, store = _check_cache(cache, table)
    device = store.device
    heads, dim = args[5:]
    check_cuda("q", q, 4, _BF16, device)
    batch, q_heads, queries, q_dim = q.shape
    if q_dim != dim or q_heads % heads or q_heads == 0:
        raise ValueError(f"q must have a multiple of {heads} heads of {dim} dimensions, got {tuple(q.shape)}")
    check_cuda("lengths", lengths, 1, _I32, device)
    if table.shape[0] != batch or lengths.shape[0] != batch:
        raise ValueError(f"table and lengths must have {batch} rows, got {table.shape[0]} and {lengths.shape[0]}")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("scale must be positive")
    _no_grad("kv8_attention", q)
    q, given = _rows(q), out is not None
    if not given:
        out = torch.empty_like(q)
        if out.stride(3) != 1 or (out.stride(0) | out.stride(1) | out.stride(2)) & 7:
            out = torch.empty(q.shape, dtype=q.dtype, device=device)
    else:
        check_cuda("out", out, 4, _BF16, device)
        check_target("out", out)
        if out.shape != q.shape:
            raise ValueError(f"out must have shape {tuple(q.shape)}, got {tuple(out.shape)}")
        if out.numel() and (out.stride(3) != 1 or (out.stride(0) | out.stride(1) | out.stride(2)) & 7
                            or out.data_ptr() & 15 or overlaps_itself(out)):
            raise ValueError("out must be 16-byte aligned, with last stride 1, the others multiples of 8 and no "
                             "broadcast dimension")
    table, lengths = table.contiguous(), lengths.contiguous()
    size = _workspace_bytes(dim, device.index)
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    launch("pasa_kv8_attention", device, q.data_ptr(), _strides(q), *args, table.data_ptr(), table.shape[1],
           lengths.data_ptr(), batch, queries, q_heads // heads, scale, out.data_ptr(), _strides(out),
           workspace.data_ptr(), size)
    if given:
        written(out)
    return out
