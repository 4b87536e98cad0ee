"""Whether the paged forward answers as a decoder's own attention does.

Names of classes and attributes cannot tell: a layer may leave its queries
unrotated, scale them by position, or rotate neighbouring pairs.  So before
``attach`` gives a decoder its paged forward, each attention module's own forward
runs on given queries, keys and values (``check_attention``), inside forwards of
the whole model on random tokens, a few at the first positions and more up to the
farthest, and what reaches its output projection is compared with the paged formula
in plain torch.
The layers meanwhile add zeros, so whatever one token still does to the tokens
behind it comes from a part of the model that the cache does not serve.
"""

from __future__ import annotations

from typing import Any, Callable

import torch
from torch import nn

_TOKENS = 24         # of a short run, and the last ones that are compared
_FAR_TOKENS = 1032   # of the run that ends at the farthest position: a window that nothing names, up to 1024, shows
_MOST_WINDOW = 4096  # longest window whose edge is looked at
_SCORE = 3.0         # standard deviation of the scores


def _most_off(dtype: torch.dtype, end: int) -> float:
    """Difference that roundings explain: 16-bit attention of such scores is off
    by 0.7 eps, and 32 bits hold the angle of position ``end`` to 2^-24 of it."""
    return max(3 * torch.finfo(dtype).eps, 2.0**-10) + end * 2.0**-24


class _Given(nn.Module):
    """Stands for a projection into queries, keys or values."""

    def __init__(self) -> None:
        super().__init__()
        self.value: torch.Tensor | None = None

    def forward(self, *args: Any, **kwargs: Any) -> torch.Tensor:
        return self.value


class _Caught(nn.Module):
    """Stands for the output projection: keeps what it gets, gives zeros."""

    def __init__(self, features: int) -> None:
        super().__init__()
        self.features = features
        self.value: torch.Tensor | None = None

    def forward(self, x: torch.Tensor, *args: Any, **kwargs: Any) -> torch.Tensor:
        self.value = x
        return x.new_zeros((*x.shape[:-1], self.features))


class _Ended(Exception):
    """The last attention module has been compared; the rest of the forward is not needed."""


def paged_formula(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, start: int, inv_freq: torch.Tensor | None, *,
                  interleaved: bool, rotary_scale: float, scale: float, window: int, last: int) -> torch.Tensor:
    """What ``paged_append`` and ``paged_attention`` give for the last tokens of
    rows that begin at position ``start``: q (B, M, heads, D), k and v (B, M,
    kv_heads, D), in 64 bits."""
    new, dim = q.shape[1], q.shape[3]
    at = torch.arange(new, device=q.device)

    def turned(x: torch.Tensor) -> torch.Tensor:
        x = x.double()
        if inv_freq is None:
            return x
        pairs = inv_freq.shape[0]
        angle = (start + at).double()[:, None] * inv_freq.detach().to(q.device, torch.float64)
        cos, sin = angle.cos()[:, None] * rotary_scale, angle.sin()[:, None] * rotary_scale
        if interleaved:
            a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
            both = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :pairs], x[..., pairs:2 * pairs]
            both = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([both, x[..., 2 * pairs:dim]], -1)

    group = q.shape[2] // k.shape[2]
    q, k = turned(q)[:, -last:], turned(k).repeat_interleave(group, 2)
    score = torch.einsum("bmhd,bnhd->bhmn", q, k) * scale
    mine = at[-last:, None]
    seen = (at[None, :] <= mine) & (at[None, :] > mine - (window or new))
    p = torch.softmax(score.masked_fill(~seen, -torch.inf), -1)
    return torch.einsum("bhmn,bnhd->bmhd", p, v.double().repeat_interleave(group, 2))


def _off(got: torch.Tensor, want: torch.Tensor) -> float:
    """Size of the difference next to what is wanted; a NaN is infinitely far."""
    want = want.double()
    off = (got.double() - want).norm() / want.norm().clamp_min(torch.finfo(torch.float32).tiny)
    return float(torch.nan_to_num(off, nan=torch.inf))


class _Probe:
    """The forward of an attention module during a run."""

    def __init__(self, module: nn.Module, forward: Any, layer: int, rotations: Callable[[], list],
                 features: tuple[int, int, int], drawn: dict) -> None:
        self.module, self.forward, self.layer, self.rotations = module, forward, layer, rotations
        self.features, self.drawn = features, drawn
        self.start, self.stop, self.seen = 0, False, False

    def draw(self, like: torch.Tensor) -> list[torch.Tensor]:
        """Queries, keys and values; the same ones for layers of the same sizes."""
        f = self.forward
        size = (_SCORE / (abs(f.scale) * f.head_dim**0.5)) ** 0.5 if f.scale else 1.0  # of a query's and a key's elements
        key = (like.shape[:2], like.dtype, like.device, self.features, size)
        if key not in self.drawn:
            g = torch.Generator().manual_seed(0)
            self.drawn.clear()
            self.drawn[key] = [torch.randn((*like.shape[:2], n), generator=g).mul_(by).to(like)
                               for n, by in zip(self.features, (size, size, 1.0))]
        return self.drawn[key]

    def __call__(self, hidden_states: torch.Tensor, *args: Any, **kwargs: Any):
        m, f = self.module, self.forward
        rows, new = hidden_states.shape[:2]
        q, k, v = self.draw(hidden_states)
        m.q_proj.value, m.k_proj.value, m.v_proj.value = q.clone(), k.clone(), v.clone()  # it may write to them
        m.o_proj.value = None
        f.original(hidden_states, *args, **kwargs)
        got, last = m.o_proj.value, min(new, _TOKENS)
        if got is None or got.numel() != q.numel():
            raise ValueError(f"attention layer {self.layer} ({type(m).__name__}) does not project its "
                             f"{q.shape[-1]} query features' attention")
        got = got.reshape(rows, new, -1, f.head_dim)[:, -last:]
        heads = [t.view(rows, new, -1, f.head_dim) for t in (q, k, v)]

        def off(interleaved: bool) -> float:
            return min(_off(got, paged_formula(*heads, self.start, inv_freq, interleaved=interleaved, rotary_scale=by,
                                               scale=f.scale, window=f.window, last=last))
                       for inv_freq, by in self.rotations())

        most = _most_off(hidden_states.dtype, self.start + new)
        mine = off(f.interleaved)
        if mine > most:
            hint = ""
            if off(not f.interleaved) <= most:
                hint = (": it rotates neighbouring pairs, pass interleaved=True" if not f.interleaved
                        else ": it rotates halves, pass interleaved=False")
            raise ValueError(f"attention layer {self.layer} ({type(m).__name__}) differs from the paged forward by "
                             f"{mine:.2g} of its size at positions {self.start + new - last} to {self.start + new - 1}{hint}")
        self.seen = True
        if self.stop:
            raise _Ended
        return torch.zeros_like(hidden_states), None


def _rotary_modules(model: nn.Module) -> list[nn.Module]:
    return [m for m in model.modules() if isinstance(getattr(m, "inv_freq", None), torch.Tensor)]


def check_attention(model: nn.Module, modules: list[nn.Module], forwards: list[Any], inv_freq: torch.Tensor,
                    rotary_scale: float, given: bool, reach: int) -> None:
    """Raises ValueError where a module of ``modules`` answers differently from
    its paged forward (of ``forwards``) at positions up to ``reach``, or where
    tokens meet outside of them.  ``given``: the frequencies are the caller's, who
    may want others than the model's; the model's own are then taken as well."""
    rotary = _rotary_modules(model)

    def rotations() -> list:
        own = [(m.inv_freq, float(getattr(m, "attention_scaling", 1.0))) for m in rotary
               if given and m.inv_freq.dim() == 1 and 2 * m.inv_freq.shape[0] <= forwards[0].head_dim]
        return [(inv_freq, rotary_scale), *own]

    embedding = (model.get_input_embeddings() if hasattr(model, "get_input_embeddings")
                 else next((m for m in model.modules() if isinstance(m, nn.Embedding)), None))
    weight = getattr(embedding, "weight", None)
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("the model has no input embeddings to check its attention with: pass check=False to go without")
    limit = getattr(getattr(modules[0], "config", None), "max_position_embeddings", None)
    reach = min(reach, limit) if isinstance(limit, int) and limit > 0 else reach
    near = min(reach, _TOKENS)
    edges = {min(f.window + 8, reach) for f in forwards if near <= f.window <= _MOST_WINDOW and f.window < reach}

    names = ("q_proj", "k_proj", "v_proj", "o_proj")
    children = [[getattr(m, n) for n in names] for m in modules]
    drawn: dict = {}
    probes = [_Probe(m, f, i, rotations, tuple(c.out_features for c in kept[:3]), drawn)
              for i, (m, f, kept) in enumerate(zip(modules, forwards, children))]
    before = [m.__dict__.get("forward") for m in modules]
    training = [(m, m.training) for m in model.modules()]
    state = [(m, dict(m.__dict__), dict(m._buffers)) for m in rotary]  # some renew their frequencies in a forward

    def run(start: int, new: int, whole: bool) -> None:
        # tokens from the middle of the vocabulary: special ones lie at its ends
        vocab = weight.shape[0]
        ids = vocab // 8 + torch.randint(0, max(vocab // 2, 1), (1, new), generator=torch.Generator().manual_seed(new))
        if whole:  # twice, apart from the first token
            ids = ids.repeat(2, 1)
            ids[1, 0] = (ids[1, 0] + 1) % vocab
        for p in probes:
            p.start, p.stop, p.seen = start, False, False
        probes[-1].stop = not whole
        at = torch.arange(start, start + new, device=weight.device)[None]
        try:
            out = model(input_ids=ids.to(weight.device), position_ids=at, use_cache=False)
        except _Ended:
            out = None
        missed = [p.layer for p in probes if not p.seen]
        if missed:
            raise ValueError(f"a forward of the model does not reach its attention layers {missed}")
        if out is None:
            return
        out = next((t for t in (getattr(out, "last_hidden_state", None), getattr(out, "logits", None), out)
                    if isinstance(t, torch.Tensor)), None)
        if out is None or out.shape[:2] != (2, new):
            return
        off = _off(out[1, 1:], out[0, 1:]) if new > 1 else 0.0
        if off > _most_off(out.dtype, new):
            raise ValueError("the model mixes its tokens outside of the attention layers that the paged forward serves")

    try:
        model.eval()
        for m, p, kept in zip(modules, probes, children):
            m.q_proj, m.k_proj, m.v_proj, m.o_proj = _Given(), _Given(), _Given(), _Caught(kept[3].out_features)
            m.forward = p
        with torch.no_grad():
            run(0, near, True)
            if reach > near:
                far = min(reach, _FAR_TOKENS)
                run(reach - far, far, False)
            for new in sorted(edges):
                run(0, new, False)
    except TypeError as e:
        raise ValueError(f"the model's attention could not be checked ({e}): pass check=False to go without") from e
    finally:
        for m, f, kept in zip(modules, before, children):
            for n, child in zip(names, kept):
                setattr(m, n, child)
            if f is None:
                m.__dict__.pop("forward", None)
            else:
                m.forward = f
        for m, flag in training:
            m.training = flag
        for m, held, buffers in state:
            m.__dict__.clear()
            m.__dict__.update(held)
            m._buffers.clear()
            m._buffers.update(buffers)
