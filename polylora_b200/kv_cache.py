"""A paged key-value cache for the wrapped decoder, and the attention that uses it.

``PagedKVCache`` owns the pages of all layers and hands them to sequences;
``PagedKVCache.batch`` takes the pages that a batch's new tokens need and returns
a ``PagedBatch``, the device tensors one forward reads.  ``PolyLoraModel.attach_kv_cache``
gives the base model's attention modules a second forward: while a PagedBatch is
installed (``PolyLoraModel.forward(..., paged=batch)``) they rotate and append
with ``paged_append`` and attend with ``paged_attention``; without one they run
as before.

Addresses do not change as sequences grow, so a decode step with its history can
be captured once and replayed (``GraphedForward(..., paged=batch)``).  The
reference has no counterpart: its forwards carry whatever cache the base model
brings.
"""

from __future__ import annotations

from contextlib import contextmanager
from contextvars import ContextVar
from dataclasses import dataclass
from typing import Any, Hashable, Iterator

import torch
import torch.nn.functional as F
from torch import nn

from .kv_check import check_attention
from .paged import paged_append, paged_attention, rotary_phases


@dataclass(frozen=True)
class PagedBatch:
    """What one forward reads: row b's new tokens are positions
    ``past_lens[b] .. past_lens[b] + new_lens[b] - 1`` of its sequence."""

    cache: "PagedKVCache"
    page_table: torch.Tensor  # (B, width) int32
    past_lens: torch.Tensor   # (B,) int32
    new_lens: torch.Tensor    # (B,) int32
    seq_lens: torch.Tensor    # (B,) int32: past + new
    max_new: int              # tokens of a row of the forward's inputs
    fresh: bool               # no row has a past (one new token a row runs alike either way)

    @property
    def rows(self) -> int:
        return self.page_table.shape[0]

    def clone(self) -> "PagedBatch":
        return PagedBatch(self.cache, self.page_table.clone(), self.past_lens.clone(), self.new_lens.clone(),
                          self.seq_lens.clone(), self.max_new, self.fresh)

    def check_copy(self, other: "PagedBatch") -> None:
        """Raises ValueError where a forward captured with this batch would not run on ``other`` as an eager one does."""
        if other.cache is not self.cache or other.max_new != self.max_new \
                or (self.max_new > 1 and other.fresh != self.fresh) or other.page_table.shape != self.page_table.shape:
            raise ValueError("a captured forward takes batches of its cache, rows, page-table width and new tokens")

    def copy_(self, other: "PagedBatch") -> None:
        """Takes another batch's tensors into this one's memory (for a captured forward)."""
        self.check_copy(other)
        for name in ("page_table", "past_lens", "new_lens", "seq_lens"):
            getattr(self, name).copy_(getattr(other, name), non_blocking=True)


_CURRENT: ContextVar[PagedBatch | None] = ContextVar("polylora_b200_paged_batch", default=None)


def get_paged_batch() -> PagedBatch | None:
    return _CURRENT.get()


@contextmanager
def use_paged_batch(batch: PagedBatch | None) -> Iterator[None]:
    token = _CURRENT.set(batch)
    try:
        yield
    finally:
        _CURRENT.reset(token)


class PagedKVCache:
    """Pages of ``page_size`` tokens for ``num_layers`` layers.

    ``k`` and ``v`` are (num_layers, num_pages, kv_heads, page_size, head_dim).
    A sequence (any hashable id) holds the pages that its tokens need; page ids
    are the same in all layers.  All methods run on the host; ``batch`` copies
    its tables with one asynchronous copy on the current stream."""

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype, device: torch.device | str) -> None:
        if min(num_layers, num_pages, page_size, num_kv_heads, head_dim) < 1:
            raise ValueError("layers, pages, page_size, heads and head_dim must be at least 1")
        self.num_layers, self.num_pages, self.page_size = num_layers, num_pages, page_size
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict[Hashable, list[int]] = {}
        self._lens: dict[Hashable, int] = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: Hashable) -> int:
        """Tokens of a sequence, those of batches already made included; 0 for an unknown one."""
        return self._lens.get(seq, 0)

    def truncate(self, seq: Hashable, length: int) -> None:
        """Drops a sequence's tokens past ``length`` (0: forgets it) and frees their pages."""
        if not 0 <= length <= self.length(seq):
            raise ValueError(f"sequence {seq!r} has {self.length(seq)} tokens, cannot keep {length}")
        if seq not in self._pages:
            return
        keep = -(-length // self.page_size)
        self._free.extend(reversed(self._pages[seq][keep:]))
        del self._pages[seq][keep:]
        self._lens[seq] = length
        if length == 0:
            del self._pages[seq], self._lens[seq]

    def free(self, seq: Hashable) -> None:
        self.truncate(seq, 0)

    def batch(self, seqs: list[Hashable], new_lens: list[int] | int = 1, max_new: int | None = None,
              width: int | None = None) -> PagedBatch:
        """Takes the pages for ``new_lens[b]`` more tokens of each sequence and
        returns the batch that appends and attends to them.  ``max_new`` (default:
        the longest of new_lens) is the width of the forward's right-padded rows,
        ``width`` (default: the most pages of a row) that of the page table, for a
        captured forward's fixed shapes.  Raises RuntimeError, with nothing taken,
        when pages run out."""
        news = [new_lens] * len(seqs) if isinstance(new_lens, int) else list(new_lens)
        if len(news) != len(seqs):
            raise ValueError("new_lens must have one entry per sequence")
        if len(set(seqs)) != len(seqs):
            raise ValueError("a batch has each sequence once: rows must not share pages that they write")
        if any(n < 0 for n in news):
            raise ValueError("new_lens must not be negative")
        longest = max(news, default=0)
        if max_new is None:
            max_new = longest
        elif max_new < longest:
            raise ValueError(f"max_new {max_new} is below the longest row, {longest}")
        past = [self.length(s) for s in seqs]
        totals = [p + n for p, n in zip(past, news)]
        need = [-(-t // self.page_size) for t in totals]
        most = max(need, default=0)
        if width is None:
            width = max(most, 1)
        elif width < max(most, 1):
            raise ValueError(f"width {width} is below the {most} pages of a row")
        more = sum(n - len(self._pages.get(s, ())) for s, n in zip(seqs, need))
        if more > len(self._free):
            raise RuntimeError(f"paged cache has {len(self._free)} free pages, the batch needs {more}")
        rows = len(seqs)
        host = torch.full((rows * (width + 3),), -1, dtype=torch.int32)  # the table, then the three lengths
        table = host[:rows * width].view(rows, width)
        for b, (s, n, t) in enumerate(zip(seqs, need, totals)):
            if t:
                pages = self._pages.setdefault(s, [])
                while len(pages) < n:
                    pages.append(self._free.pop())
                self._lens[s] = t
                table[b, :n] = torch.tensor(pages, dtype=torch.int32)
        host[rows * width:] = torch.tensor(past + news + totals, dtype=torch.int32)
        device = self.k.device
        dev = host.pin_memory().to(device, non_blocking=True) if device.type == "cuda" else host
        lens = dev[rows * width:].view(3, rows)
        return PagedBatch(self, dev[:rows * width].view(rows, width), lens[0], lens[1], lens[2], max_new, not any(past))


_MOST_ROWS = 1 << 20  # of a call of paged_attention


class _PagedAttentionForward:
    """The forward of an attention module under a PagedBatch."""

    def __init__(self, module: nn.Module, original, cache: PagedKVCache, layer: int, phases: torch.Tensor | None,
                 interleaved: bool, rotary_scale: float) -> None:
        self.module, self.original, self.cache, self.layer = module, original, cache, layer
        self.phases, self.interleaved, self.rotary_scale = phases, interleaved, rotary_scale
        self.head_dim = int(module.head_dim)
        self.scale = float(getattr(module, "scaling", self.head_dim**-0.5))
        self.window = _window(module)

    def __call__(self, hidden_states: torch.Tensor, *args: Any, **kwargs: Any):
        batch = get_paged_batch()
        if batch is None:
            return self.original(hidden_states, *args, **kwargs)
        if batch.cache is not self.cache:
            raise ValueError("the batch belongs to another cache than the one attached")
        rows, new = hidden_states.shape[:2]
        if (rows, new) != (batch.rows, batch.max_new):
            raise ValueError(f"paged batch of {batch.rows} x {batch.max_new} tokens, inputs of {rows} x {new}")
        m, d = self.module, self.head_dim
        q, k, v = (proj(hidden_states).view(rows, new, -1, d) for proj in (m.q_proj, m.k_proj, m.v_proj))
        kc, vc = self.cache.k[self.layer], self.cache.v[self.layer]
        prompt = new > 1 and batch.fresh
        if self.phases is not None and self.phases.device != q.device:
            self.phases = self.phases.to(q.device)
        q, k = paged_append(q, k, v, kc, vc, batch.page_table, batch.past_lens, batch.new_lens, phases=self.phases,
                            interleaved=self.interleaved, rotary_scale=self.rotary_scale, return_keys=prompt)
        if prompt:
            out = self._prompt(q, k, v)
        elif new == 1:
            out = paged_attention(q[:, 0], kc, vc, batch.page_table, batch.seq_lens, scale=self.scale, window=self.window)
        else:  # a few tokens after a history: each is a row that sees the tokens up to itself
            step = torch.arange(new, dtype=torch.int32, device=q.device)
            live = step < batch.new_lens[:, None]
            lens = torch.where(live, batch.past_lens[:, None] + step + 1, 0).view(-1)
            q = q.view(rows * new, -1, d)
            out = torch.empty_like(q)
            for first in range(0, rows * new, _MOST_ROWS):
                part = slice(first, min(first + _MOST_ROWS, rows * new))
                row = torch.arange(part.start, part.stop, device=q.device) // new
                paged_attention(q[part], kc, vc, batch.page_table[row], lens[part], scale=self.scale, window=self.window,
                                out=out[part])
        return m.o_proj(out.reshape(rows, new, -1)), None

    def _prompt(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """Causal attention among a fresh batch's own tokens; right padding is behind them."""
        new = q.shape[1]
        mask = None
        if 0 < self.window < new:
            at = torch.arange(new, device=q.device)
            mask = (at[None, :] <= at[:, None]) & (at[None, :] > at[:, None] - self.window)
        out = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), attn_mask=mask,
                                             is_causal=mask is None, scale=self.scale,
                                             enable_gqa=q.shape[2] != k.shape[2])
        return out.transpose(1, 2)


def _window(module: nn.Module) -> int:
    """Tokens that a layer's attention reaches back (0: all)."""
    config = getattr(module, "config", None)
    window = getattr(module, "sliding_window", None) or getattr(config, "sliding_window", None)
    types = getattr(config, "layer_types", None)
    if types is not None and types[module.layer_idx] != "sliding_attention":
        return 0
    return int(window or 0)


def _check_attention(module: nn.Module) -> None:
    """Refuses attention that ``_PagedAttentionForward`` would answer differently:
    it projects, rotates, and takes a causal softmax of the scaled products."""
    config = getattr(module, "config", None)
    own = [n for n, _ in module.named_parameters(recurse=False)] + [n for n, _ in module.named_buffers(recurse=False)]
    if own:  # such as learned attention sinks
        raise ValueError(f"an attention module has parameters of its own: {', '.join(own)}")
    if not getattr(module, "is_causal", True):
        raise ValueError("an attention module is not causal")
    if not getattr(module, "use_rope", True):
        raise ValueError("an attention module does not rotate its queries and keys")
    for name in ("attn_logit_softcapping", "clip_qkv"):
        if getattr(module, name, None) is not None or getattr(config, name, None) is not None:
            raise ValueError(f"an attention module has {name}")
    types = getattr(config, "layer_types", None)
    if types is not None and types[module.layer_idx] not in ("full_attention", "sliding_attention"):
        raise ValueError(f"an attention layer is of type {types[module.layer_idx]!r}")


_PROJECTIONS = {"q_proj", "k_proj", "v_proj", "o_proj"}


def attention_modules(model: nn.Module) -> list[nn.Module]:
    """The model's attention modules, in order: those whose children are the
    query, key, value and output projections alone."""
    return [m for m in model.modules() if {n for n, _ in m.named_children()} == _PROJECTIONS and hasattr(m, "head_dim")]


def _rotation(model: nn.Module) -> tuple[torch.Tensor, float]:
    """(inv_freq, scale of sines and cosines) of the model's rotary embedding."""
    found = [m for m in model.modules() if isinstance(getattr(m, "inv_freq", None), torch.Tensor)]
    if len(found) != 1 or found[0].inv_freq.dim() != 1:
        raise ValueError("the model has not one rotary embedding with inv_freq: pass inv_freq")
    kind = getattr(found[0], "rope_type", "default")
    if kind not in ("default", "linear", "llama3", "yarn"):
        raise ValueError(f"rotary embedding of type {kind!r} changes its frequencies with the length")
    return found[0].inv_freq, float(getattr(found[0], "attention_scaling", 1.0))


def attach(model: nn.Module, cache: PagedKVCache, inv_freq: torch.Tensor | None = None,
           rotary_scale: float | None = None, interleaved: bool = False, check: bool = True) -> None:
    """Gives the model's attention modules their paged forward (see
    ``PolyLoraModel.attach_kv_cache``)."""
    modules = attention_modules(model)
    if len(modules) != cache.num_layers:
        raise ValueError(f"the model has {len(modules)} attention modules, the cache {cache.num_layers} layers")
    _, _, kv_heads, _, head_dim = cache.k.shape
    for m in modules:
        _check_attention(m)
        if int(m.head_dim) != head_dim or m.k_proj.out_features != kv_heads * head_dim:
            raise ValueError(f"an attention module has {m.k_proj.out_features} key features in heads of {m.head_dim}, "
                             f"the cache {kv_heads} heads of {head_dim}")
    given = inv_freq is not None
    if not given:
        inv_freq, scale = _rotation(model)
    else:
        scale = 1.0
    if rotary_scale is None:
        rotary_scale = scale
    phases = rotary_phases(inv_freq)
    forwards = []
    for layer, m in enumerate(modules):
        original = m.forward.original if isinstance(m.forward, _PagedAttentionForward) else m.forward
        forwards.append(_PagedAttentionForward(m, original, cache, layer, phases, interleaved, rotary_scale))
    if check:
        check_attention(model, modules, forwards, inv_freq, rotary_scale, given, cache.num_pages * cache.page_size)
    for m, f in zip(modules, forwards):
        m.forward = f


__all__ = ["PagedBatch", "PagedKVCache", "get_paged_batch", "use_paged_batch"]
