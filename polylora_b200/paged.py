"""Paged key-value cache operators over the C-ABI library.

* :func:`paged_append` — rotates a batch's new queries and keys by their
  positions and writes keys and values to the rows' pages.
* :func:`paged_attention` — attention of one new token per row over its pages.
* :func:`rotary_phases` — a model's rotation frequencies in the form the
  append takes, once per model.

The cache of a layer is two tensors (num_pages, kv_heads, page_size, head_dim);
position p of row b is slot ``p % page_size`` of page
``page_table[b, p // page_size]``.  The reference has no counterpart: it wraps
models that bring their own caches.
"""

from __future__ import annotations

import functools
import math

import torch
from torch.autograd import forward_ad

from . import _native
from .sgmv import _as, _require_cuda, dtype_code


def rotary_phases(inv_freq: torch.Tensor) -> torch.Tensor:
    """``inv_freq`` (pairs,) in radians per position as 64-bit fractions of a
    turn (int64, same device): position * phase mod 2^64 is the exact angle."""
    if inv_freq.dim() != 1 or not inv_freq.is_floating_point():
        raise ValueError("inv_freq must be a 1D floating-point tensor")
    host = inv_freq.detach().double().cpu()
    if not bool(torch.isfinite(host).all()):
        raise ValueError("inv_freq must be finite")
    turn = torch.remainder(host / (2 * math.pi), 1.0) * 2.0**32
    high = turn.floor()
    low = ((turn - high) * 2.0**32).round()
    return ((high.to(torch.int64) << 32) + low.to(torch.int64)).to(inv_freq.device)  # mod 2^64


def _no_grad(*tensors: torch.Tensor | None) -> None:
    """Refuses tensors whose gradients or tangents would be lost without a word."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("the paged-cache and logit operators have no gradient: call them under torch.no_grad()")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("the paged-cache and logit operators have no gradient, and a tensor carries a tangent")


def _same_device(index: int, *tensors: torch.Tensor) -> None:
    """All on CUDA device ``index``.  (Ordinals: a decode step's kernels take a
    few microseconds, and comparing torch.device objects would take one.)"""
    if index < 0:
        _require_cuda(*tensors)
    for t in tensors:
        if t.get_device() != index:
            raise ValueError(f"tensors on different devices: cuda:{index} and {t.device}")


def _strides(t: torch.Tensor) -> tuple[int, ...]:
    """Strides, 0 for dimensions of one."""
    return tuple([st if n > 1 else 0 for n, st in zip(t.shape, t.stride())])


def _heads(t: torch.Tensor) -> tuple[torch.Tensor, tuple[int, ...], int]:
    """``t`` with dense last dimension and 16-byte aligned rows (a copy where
    it has neither), its strides and its address."""
    ptr, st, size = t.data_ptr(), t.stride(), t.element_size()
    if st[-1] == 1 and not ((st[0] | st[1] | st[-2]) * size | ptr) & 15:  # the rule, with any dimensions of one
        return t, st, ptr
    st, vec = _strides(t), 16 // size
    if (t.shape[-1] > 1 and st[-1] != 1) or any([s % vec for s in st[:-1]]) or ptr % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        st, ptr = _strides(t), t.data_ptr()
    return t, st, ptr


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, rows: int, dim: int,
                 dtype: torch.dtype) -> tuple[int, int, int, int, int, int, int]:
    """(num_pages, kv_heads, page_size, k page stride, v page stride, page-table row stride, max_pages)."""
    shape = k_cache.shape
    if len(shape) != 4 or shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must both be (num_pages, kv_heads, page_size, head_dim)")
    pages, kv_heads, size, d = shape
    if d != dim:
        raise ValueError(f"head_dim mismatch: tokens={dim}, cache={d}")
    if k_cache.dtype is not dtype or v_cache.dtype is not dtype:
        raise TypeError(f"dtype mismatch: tokens={dtype}, k_cache={k_cache.dtype}, v_cache={v_cache.dtype}")
    page = kv_heads * size * d
    k_page = v_page = page
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        inner = (size * d, d, 1)
        for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
            if any([st != want for n, st, want in zip(c.shape[1:], c.stride()[1:], inner) if n > 1]):
                raise ValueError(f"{name} pages must be contiguous")
        if pages > 1:
            k_page, v_page = k_cache.stride(0), v_cache.stride(0)
    table = page_table.shape
    if page_table.dtype is not torch.int32 or len(table) != 2 or table[0] != rows:
        raise ValueError(f"page_table must be int32 ({rows}, max_pages)")
    row, step = page_table.stride()
    if step != 1 and table[1] > 1:
        raise ValueError("page_table rows must be contiguous")
    return pages, kv_heads, size, k_page, v_page, row if rows > 1 else table[1], table[1]


def _lens(t: torch.Tensor, rows: int, name: str) -> torch.Tensor:
    if t.dim() != 1 or t.shape[0] != rows:
        raise ValueError(f"{name} must have shape ({rows},), got {tuple(t.shape)}")
    return _as(t, torch.int32)


# Sizes alone decide it; asking the library takes a microsecond of a call whose kernel takes seven.
@functools.lru_cache(maxsize=1024)
def _attention_workspace(rows: int, heads: int, kv_heads: int, dim: int, size: int, max_pages: int, window: int,
                         dtype: int) -> int:
    return _native.load().plora_paged_attention_workspace(rows, heads, kv_heads, dim, size, max_pages, window, dtype)


# The current stream's raw handle: a Stream object costs 2 us of a call whose kernel takes less than 3.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch.cuda.current_device


def paged_append(
    q: torch.Tensor | None,
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    past_lens: torch.Tensor,
    new_lens: torch.Tensor | None = None,
    *,
    phases: torch.Tensor | None = None,
    interleaved: bool = False,
    rotary_scale: float = 1.0,
    return_keys: bool = False,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """Appends new tokens to the cache, rotated by their positions.

    q (B, M, heads, D) or None, k and v (B, M, kv_heads, D); row b's first
    ``new_lens[b]`` tokens (None: all M) take the positions from
    ``past_lens[b]`` on.  ``phases`` (:func:`rotary_phases`) rotates the first
    2 * len(phases) elements of each query and key head (None: no rotation), in
    halves or as neighbouring pairs (``interleaved``), with sines and cosines
    times ``rotary_scale``.  k_cache and v_cache are updated in place.  Returns
    the rotated queries and, with ``return_keys``, the rotated keys (padded
    tokens zero); None for what was not given or asked for.  Rows of one call
    must not write to the same page, nor keys and values to the same memory (their
    pages may interleave)."""
    dev = k.get_device()
    if dev < 0 or not (v.get_device() == k_cache.get_device() == v_cache.get_device() == page_table.get_device()
                       == past_lens.get_device() == dev):
        _same_device(dev, k, v, k_cache, v_cache, page_table, past_lens)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return paged_append(q, k, v, k_cache, v_cache, page_table, past_lens, new_lens, phases=phases,
                                interleaved=interleaved, rotary_scale=rotary_scale, return_keys=return_keys)
    _no_grad(q, k, v, k_cache, v_cache)
    shape, dtype = k.shape, k.dtype
    if len(shape) != 4 or v.shape != shape:
        raise ValueError("q must be (B, M, heads, D), k and v (B, M, kv_heads, D)")
    rows, new, kv_heads, dim = shape
    if v.dtype is not dtype:
        raise TypeError("q, k and v must share one dtype")
    pages, ckv, size, k_page, v_page, table_row, max_pages = _check_cache(k_cache, v_cache, page_table, rows, dim, dtype)
    if ckv != kv_heads:
        raise ValueError(f"kv_heads mismatch: k={kv_heads}, cache={ckv}")
    past = _lens(past_lens, rows, "past_lens")
    news_ptr = phases_ptr = q_ptr = q_out_ptr = k_out_ptr = pairs = heads = 0
    q_out = k_out = None
    qs = (0, 0, 0)
    if new_lens is not None:
        if new_lens.get_device() != dev:
            _same_device(dev, new_lens)
        new_lens = _lens(new_lens, rows, "new_lens")
        news_ptr = new_lens.data_ptr()
    if phases is not None:
        if phases.get_device() != dev:
            _same_device(dev, phases)
        if phases.dim() != 1 or phases.dtype is not torch.int64:
            raise ValueError("phases must be the int64 tensor of rotary_phases()")
        pairs = phases.shape[0]
        phases = phases.contiguous()
        phases_ptr = phases.data_ptr() if pairs else 0
    if q is not None:
        if q.get_device() != dev:
            _same_device(dev, q)
        if q.dtype is not dtype:
            raise TypeError("q, k and v must share one dtype")
        shape = q.shape
        if len(shape) != 4 or shape[0] != rows or shape[1] != new or shape[3] != dim:
            raise ValueError("q must be (B, M, heads, D), k and v (B, M, kv_heads, D)")
        heads = shape[2]
        q_out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
        q_out_ptr = q_out.data_ptr()
        q, qs, q_ptr = _heads(q)
    k, ks, k_ptr = _heads(k)
    v, vs, v_ptr = _heads(v)
    if return_keys:
        k_out = k.new_empty((rows, new, kv_heads, dim))
        k_out_ptr = k_out.data_ptr()
    args = _native.PAGED_APPEND_ARGS.pack(
        k_cache.data_ptr(), v_cache.data_ptr(), k_page, v_page, page_table.data_ptr(), table_row, rows, heads, kv_heads,
        dim, size, pages, max_pages, dtype_code(dtype),
        q_ptr, qs[0], qs[1], qs[2], k_ptr, ks[0], ks[1], ks[2], v_ptr, vs[0], vs[1], vs[2],
        q_out_ptr, k_out_ptr, past.data_ptr(), news_ptr, phases_ptr, pairs, interleaved, new, rotary_scale,
    )
    status = _native.load().plora_paged_append(args, _raw_stream(dev))
    if status:
        _native.check("plora_paged_append", status)
    return q_out, k_out


def paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    scale: float | None = None,
    window: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of one token per row, q (B, heads, D), over the row's first
    ``seq_lens[b]`` cached tokens (the last ``window`` of them if window > 0).
    ``scale`` defaults to D ** -0.5; rows without tokens give zeros.  Heads may
    be any multiple of the cache's kv_heads."""
    dev = q.get_device()
    if dev < 0 or not (k_cache.get_device() == v_cache.get_device() == page_table.get_device() == seq_lens.get_device()
                       == dev):
        _same_device(dev, q, k_cache, v_cache, page_table, seq_lens)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return paged_attention(q, k_cache, v_cache, page_table, seq_lens, scale=scale, window=window, out=out)
    _no_grad(q, k_cache, v_cache)
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3:
        raise ValueError("q must be (B, heads, D)")
    rows, heads, dim = shape
    pages, kv_heads, size, k_page, v_page, table_row, max_pages = _check_cache(k_cache, v_cache, page_table, rows, dim,
                                                                               dtype)
    if heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} heads over {kv_heads} kv heads")
    lens = _lens(seq_lens, rows, "seq_lens")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    elif out.shape != shape or out.dtype is not dtype or out.get_device() != dev or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape, dtype and device")
    q, qs, q_ptr = _heads(q)
    code, lib = dtype_code(dtype), _native.load()
    ws_bytes = _attention_workspace(rows, heads, kv_heads, dim, size, max_pages, window, code)
    ws = lens.new_empty(ws_bytes // 4) if ws_bytes else None
    args = _native.PAGED_ATTENTION_ARGS.pack(
        k_cache.data_ptr(), v_cache.data_ptr(), k_page, v_page, page_table.data_ptr(), table_row, rows, heads, kv_heads,
        dim, size, pages, max_pages, code,
        q_ptr, qs[0], qs[1], lens.data_ptr(), out.data_ptr(), dim**-0.5 if scale is None else scale, window,
        ws.data_ptr() if ws_bytes else 0, ws_bytes,
    )
    status = lib.plora_paged_attention(args, _raw_stream(dev))
    if status:
        _native.check("plora_paged_attention", status)
    return out
