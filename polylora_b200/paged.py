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

import math

import torch

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
    turns = [round(math.ldexp(math.fmod(f, 2 * math.pi) / (2 * math.pi), 64)) for f in host.tolist()]
    signed = [((t + (1 << 63)) % (1 << 64)) - (1 << 63) for t in turns]
    return torch.tensor(signed, dtype=torch.int64).to(inv_freq.device)


def _no_grad(*tensors: torch.Tensor | None) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("the paged-cache and logit operators have no gradient: call them under torch.no_grad()")


def _heads(t: torch.Tensor) -> tuple[torch.Tensor, tuple[int, ...]]:
    """``t`` with dense last dimension and 16-byte aligned rows (a copy where
    it has neither) and its strides, 0 for dimensions of one."""
    vec = 16 // t.element_size()
    if t.is_contiguous() and t.shape[-1] % vec == 0:
        st = t.stride() if 1 not in t.shape else _strides(t)
    else:
        st = _strides(t)
        if (t.shape[-1] > 1 and st[-1] != 1) or any(s % vec for s in st[:-1]):
            t = t.contiguous()
            st = _strides(t)
    if t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        st = _strides(t)
    return t, st


def _strides(t: torch.Tensor) -> tuple[int, ...]:
    return tuple([st if n > 1 else 0 for n, st in zip(t.shape, t.stride())])


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, rows: int, dim: int,
                 dtype: torch.dtype) -> tuple[int, int, int, int, int]:
    """(num_pages, kv_heads, page_size, k page stride, v page stride)."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must both be (num_pages, kv_heads, page_size, head_dim)")
    pages, kv_heads, size, d = k_cache.shape
    if d != dim:
        raise ValueError(f"head_dim mismatch: tokens={dim}, cache={d}")
    if not (k_cache.dtype == v_cache.dtype == dtype):
        raise TypeError(f"dtype mismatch: tokens={dtype}, k_cache={k_cache.dtype}, v_cache={v_cache.dtype}")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        inner = (size * d, d, 1)
        for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
            if any(st != want for n, st, want in zip(c.shape[1:], c.stride()[1:], inner) if n > 1):
                raise ValueError(f"{name} pages must be contiguous")
    if page_table.dim() != 2 or page_table.shape[0] != rows or page_table.dtype != torch.int32:
        raise ValueError(f"page_table must be int32 ({rows}, max_pages)")
    if page_table.shape[1] > 1 and page_table.stride(1) != 1:
        raise ValueError("page_table rows must be contiguous")
    page = kv_heads * size * d
    return (pages, kv_heads, size, k_cache.stride(0) if pages > 1 else page,
            v_cache.stride(0) if pages > 1 else page)


def _lens(t: torch.Tensor, rows: int, name: str) -> torch.Tensor:
    if t.dim() != 1 or t.shape[0] != rows:
        raise ValueError(f"{name} must have shape ({rows},), got {tuple(t.shape)}")
    return _as(t, torch.int32)


def _call(dev: torch.device, func: str, *args: object) -> None:
    """The entry point on the device's current stream, with the device current."""
    index = dev.index
    # the raw handle: a Stream object costs 2 us of a call whose kernel takes less than 3
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch.cuda.current_device():
        _native.call(func, *args, stream)
    else:
        with torch.cuda.device(index):
            _native.call(func, *args, stream)


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
    must not write to the same page."""
    dev = _require_cuda(k, v, k_cache, v_cache, page_table, past_lens,
                        *[t for t in (q, new_lens, phases) if t is not None])
    _no_grad(q, k, v)
    if k.dim() != 4 or v.shape != k.shape or (q is not None and (q.dim() != 4 or q.shape[:2] != k.shape[:2]
                                                                 or q.shape[3] != k.shape[3])):
        raise ValueError("q must be (B, M, heads, D), k and v (B, M, kv_heads, D)")
    if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise TypeError("q, k and v must share one dtype")
    rows, new, kv_heads, dim = k.shape
    pages, ckv, size, k_page, v_page = _check_cache(k_cache, v_cache, page_table, rows, dim, k.dtype)
    if ckv != kv_heads:
        raise ValueError(f"kv_heads mismatch: k={kv_heads}, cache={ckv}")
    heads = q.shape[2] if q is not None else 0
    past = _lens(past_lens, rows, "past_lens")
    news = _lens(new_lens, rows, "new_lens") if new_lens is not None else None
    pairs = 0
    if phases is not None:
        if phases.dim() != 1 or phases.dtype != torch.int64:
            raise ValueError("phases must be the int64 tensor of rotary_phases()")
        pairs = phases.shape[0]
        phases = phases.contiguous()
    kc, ks = _heads(k)
    vc, vs = _heads(v)
    qc, qs = _heads(q) if q is not None else (None, (0, 0, 0))
    q_out = k.new_empty((rows, new, heads, dim)) if q is not None else None
    k_out = k.new_empty((rows, new, kv_heads, dim)) if return_keys else None
    _call(
        dev, "plora_paged_append",
        qc.data_ptr() if qc is not None else 0, qs[0], qs[1], qs[2], kc.data_ptr(), ks[0], ks[1], ks[2],
        vc.data_ptr(), vs[0], vs[1], vs[2], q_out.data_ptr() if q_out is not None else 0,
        k_out.data_ptr() if k_out is not None else 0, k_cache.data_ptr(), v_cache.data_ptr(), k_page, v_page,
        page_table.data_ptr(), page_table.stride(0) if rows > 1 else page_table.shape[1], past.data_ptr(),
        news.data_ptr() if news is not None else 0, phases.data_ptr() if pairs else 0, pairs, int(interleaved),
        rotary_scale, rows, new, heads, kv_heads, dim, size, pages, page_table.shape[1], dtype_code(k.dtype),
    )
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
    dev = _require_cuda(q, k_cache, v_cache, page_table, seq_lens)
    _no_grad(q)
    if q.dim() != 3:
        raise ValueError("q must be (B, heads, D)")
    rows, heads, dim = q.shape
    pages, kv_heads, size, k_page, v_page = _check_cache(k_cache, v_cache, page_table, rows, dim, q.dtype)
    if heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} heads over {kv_heads} kv heads")
    lens = _lens(seq_lens, rows, "seq_lens")
    if out is None:
        out = q.new_empty((rows, heads, dim))
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError("out must be a contiguous tensor of q's shape, dtype and device")
    qc, qs = _heads(q)
    code = dtype_code(q.dtype)
    ws_bytes = _native.load().plora_paged_attention_workspace(rows, heads, kv_heads, dim, code)
    ws = lens.new_empty(max(ws_bytes, 256) // 4)
    _call(
        dev, "plora_paged_attention",
        qc.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), k_page, v_page, page_table.data_ptr(),
        page_table.stride(0) if rows > 1 else page_table.shape[1], lens.data_ptr(), out.data_ptr(),
        dim**-0.5 if scale is None else scale, window, rows, heads, kv_heads, dim, size, pages, page_table.shape[1],
        code, ws.data_ptr(), ws_bytes,
    )
    return out
