"""Each row's own rules on its logits: penalties, biases and masks.

As every row of a batch picks its own adapter, every row carries its own
sampling rules: :class:`LogitRules` holds them as device tensors and
:func:`apply_logit_rules` applies all of them in one pass over the logits.
The reference has no counterpart (it ends at the base model's output).
"""

from __future__ import annotations

import functools
from dataclasses import dataclass

import torch

from . import _native
from .paged import _current_device, _no_grad, _raw_stream, _same_device
from .sgmv import dtype_code


@dataclass
class LogitRules:
    """Rules of a batch of B rows; None leaves a rule out.

    ``tokens`` (B, L) int32 or int64 with the first ``token_lens[b]`` (None: L)
    of each row its history, of which the first ``prompt_lens[b]`` (None: 0)
    are the prompt.  For a token of the history, x -> x / r where positive, else
    x * r, with r = ``repetition_penalty[b]``; for one that the answer (the
    history past the prompt) holds n > 0 times, x -> x - n *
    ``frequency_penalty[b]`` - ``presence_penalty[b]``.  Then
    ``bias_values[b, j]`` is added to token ``bias_tokens[b, j]`` (ids outside the
    vocabulary, such as -1 for padding, are skipped, as in ``tokens``; biases of
    one token add up), and tokens whose bit t % 32 of ``allowed[b, t // 32]``
    (int32) is 0 become -inf.
    """

    tokens: torch.Tensor | None = None
    token_lens: torch.Tensor | None = None
    prompt_lens: torch.Tensor | None = None
    repetition_penalty: torch.Tensor | None = None
    presence_penalty: torch.Tensor | None = None
    frequency_penalty: torch.Tensor | None = None
    bias_tokens: torch.Tensor | None = None
    bias_values: torch.Tensor | None = None
    allowed: torch.Tensor | None = None

    def clone(self) -> "LogitRules":
        return LogitRules(**{k: v.clone() if v is not None else None for k, v in vars(self).items()})

    def check_copy(self, other: "LogitRules") -> None:
        """Raises ValueError where ``copy_`` would not take ``other``'s values as they are."""
        for name, mine in vars(self).items():
            theirs = getattr(other, name)
            if (mine is None) != (theirs is None) or (mine is not None and mine.shape != theirs.shape):
                raise ValueError(f"{name}: a captured call takes rules of the same kinds and shapes")
            # what the operator would convert too may be; a token id or a mask may not lose bits
            if mine is not None and mine.dtype is not _TYPES.get(name) \
                    and torch.promote_types(mine.dtype, theirs.dtype) is not mine.dtype:
                raise ValueError(f"{name}: captured as {mine.dtype}, which does not hold every {theirs.dtype}")

    def copy_(self, other: "LogitRules") -> None:
        """Takes another's values into this one's memory (for a captured call);
        where one of them is refused, none is taken."""
        self.check_copy(other)
        for name, mine in vars(self).items():
            if mine is not None:
                mine.copy_(getattr(other, name), non_blocking=True)


# What the operator converts lengths and values to.
_TYPES = {"token_lens": torch.int32, "prompt_lens": torch.int32, "repetition_penalty": torch.float32,
          "presence_penalty": torch.float32, "frequency_penalty": torch.float32, "bias_values": torch.float32}


def _matrix(t: torch.Tensor, dev: int, rows: int, name: str) -> torch.Tensor:
    """A (rows, n) list with dense rows (a copy where they are not)."""
    if t.get_device() != dev:
        _same_device(dev, t)
    shape = t.shape
    if len(shape) != 2 or shape[0] != rows:
        raise ValueError(f"{name} must be 2D with {rows} rows, got {tuple(shape)}")
    return t if shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _vector(t: torch.Tensor, dev: int, rows: int, dtype: torch.dtype, name: str) -> torch.Tensor:
    """One dense value of ``dtype`` per row."""
    if t.get_device() != dev:
        _same_device(dev, t)
    if t.dim() != 1 or t.shape[0] != rows:
        raise ValueError(f"{name} must have shape ({rows},), got {tuple(t.shape)}")
    return t if t.dtype is dtype and t.is_contiguous() else t.to(dtype).contiguous()


@functools.lru_cache(maxsize=1024)  # sizes alone decide it
def _workspace(rows: int, vocab: int, history: int, biases: int) -> int:
    return _native.load().plora_logit_rules_workspace(rows, vocab, history, biases)


def apply_logit_rules(logits: torch.Tensor, rules: LogitRules, out: torch.Tensor | None = None) -> torch.Tensor:
    """``rules`` on logits (B, V), computed in fp32 and rounded once to the
    logits' dtype; into ``out`` (``logits``, or memory of its own) or a new tensor."""
    dev = logits.get_device()
    if dev < 0:
        _same_device(dev, logits)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return apply_logit_rules(logits, rules, out)
    _no_grad(logits, rules.repetition_penalty, rules.presence_penalty, rules.frequency_penalty, rules.bias_values)
    if logits.dim() != 2:
        raise ValueError("logits must be (B, V)")
    rows, vocab = logits.shape
    row, step = logits.stride()
    if step != 1 and vocab > 1:
        raise ValueError("logits rows must be contiguous")
    if out is None:
        out = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty((rows, vocab))
    elif out is not logits and (out.shape != logits.shape or out.dtype is not logits.dtype or out.get_device() != dev
                                or (vocab > 1 and out.stride(1) != 1)):
        raise ValueError("out must have the logits' shape, dtype and device, with contiguous rows")
    lens, prompt, rep, pres, freq = (rules.token_lens, rules.prompt_lens, rules.repetition_penalty,
                                     rules.presence_penalty, rules.frequency_penalty)
    tokens, bias_tokens, bias_values, allowed = rules.tokens, rules.bias_tokens, rules.bias_values, rules.allowed
    width = None
    history = biases = token_row = bias_row = value_row = mask_row = 0
    lens_ptr = prompt_ptr = rep_ptr = pres_ptr = freq_ptr = 0
    if tokens is not None:
        width = tokens.dtype
        if width is not torch.int64 and width is not torch.int32:
            raise TypeError(f"tokens must be int32 or int64, got {width}")
        tokens = _matrix(tokens, dev, rows, "tokens")
        history = tokens.shape[1]
        if lens is not None:
            lens = _vector(lens, dev, rows, torch.int32, "token_lens")
            lens_ptr = lens.data_ptr()
        if prompt is not None:
            prompt = _vector(prompt, dev, rows, torch.int32, "prompt_lens")
            prompt_ptr = prompt.data_ptr()
        if rep is not None:
            rep = _vector(rep, dev, rows, torch.float32, "repetition_penalty")
            rep_ptr = rep.data_ptr()
        if pres is not None:
            pres = _vector(pres, dev, rows, torch.float32, "presence_penalty")
            pres_ptr = pres.data_ptr()
        if freq is not None:
            freq = _vector(freq, dev, rows, torch.float32, "frequency_penalty")
            freq_ptr = freq.data_ptr()
    elif not (lens is prompt is rep is pres is freq is None):
        raise ValueError("penalties and lengths need tokens")
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias_tokens and bias_values go together")
    if bias_tokens is not None:
        if bias_tokens.dtype is not torch.int64 and bias_tokens.dtype is not torch.int32:
            raise TypeError(f"bias_tokens must be int32 or int64, got {bias_tokens.dtype}")
        if bias_tokens.shape != bias_values.shape:
            raise ValueError("bias_tokens and bias_values must have one shape")
        bias_tokens = _matrix(bias_tokens, dev, rows, "bias_tokens")
        if width is not None and bias_tokens.dtype is not width:  # both as the wider: narrowing could alias ids
            tokens, bias_tokens = tokens.to(torch.int64), bias_tokens.to(torch.int64)
        width = bias_tokens.dtype
        if bias_values.dtype is not torch.float32:
            bias_values = bias_values.to(torch.float32)
        bias_values = _matrix(bias_values, dev, rows, "bias_values")
        biases, bias_row, value_row = bias_tokens.shape[1], bias_tokens.stride(0), bias_values.stride(0)
    if tokens is not None:
        token_row = tokens.stride(0)
    if allowed is not None:
        if allowed.dtype is not torch.int32 or allowed.dim() != 2 or allowed.shape[1] < (vocab + 31) // 32:
            raise ValueError(f"allowed must be int32 ({rows}, at least {(vocab + 31) // 32})")
        allowed = _matrix(allowed, dev, rows, "allowed")
        mask_row = allowed.stride(0)
    lib = _native.load()
    ws_bytes = _workspace(rows, vocab, history, biases)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=logits.device) if ws_bytes else None
    args = _native.LOGIT_RULES_ARGS.pack(
        logits.data_ptr(), row if rows > 1 else vocab, out.data_ptr(), out.stride(0) if rows > 1 else vocab, rows, vocab,
        dtype_code(logits.dtype), tokens.data_ptr() if tokens is not None else 0, token_row, history, lens_ptr, prompt_ptr,
        rep_ptr, pres_ptr, freq_ptr, bias_tokens.data_ptr() if biases else 0, bias_row,
        bias_values.data_ptr() if biases else 0, value_row, biases, allowed.data_ptr() if allowed is not None else 0,
        mask_row, 4 if width is torch.int32 else 8, ws.data_ptr() if ws_bytes else 0, ws_bytes,
    )
    status = lib.plora_logit_rules(args, _raw_stream(dev))
    if status:
        _native.check("plora_logit_rules", status)
    return out
