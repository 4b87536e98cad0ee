"""Each row's own rules on its logits: penalties, biases and masks.

As every row of a batch picks its own adapter, every row carries its own
sampling rules: :class:`LogitRules` holds them as device tensors and
:func:`apply_logit_rules` applies all of them in one pass over the logits.
The reference has no counterpart (it ends at the base model's output).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _native
from .paged import _current_device, _no_grad, _raw_stream, _same_device
from .sgmv import _as, dtype_code


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

    def copy_(self, other: "LogitRules") -> None:
        """Takes another's values into this one's memory (for a captured call)."""
        for name, mine in vars(self).items():
            theirs = getattr(other, name)
            if (mine is None) != (theirs is None) or (mine is not None and mine.shape != theirs.shape):
                raise ValueError(f"{name}: a captured call takes rules of the same kinds and shapes")
            if mine is not None:
                mine.copy_(theirs, non_blocking=True)

    def tensors(self) -> list[torch.Tensor]:
        every = (self.tokens, self.token_lens, self.prompt_lens, self.repetition_penalty, self.presence_penalty,
                 self.frequency_penalty, self.bias_tokens, self.bias_values, self.allowed)
        return [t for t in every if t is not None]


def _rows_of(t: torch.Tensor, rows: int, name: str) -> torch.Tensor:
    if t.dim() != 2 or t.shape[0] != rows:
        raise ValueError(f"{name} must be 2D with {rows} rows, got {tuple(t.shape)}")
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _per_row(t: torch.Tensor | None, rows: int, dtype: torch.dtype, name: str) -> torch.Tensor | None:
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != rows:
        raise ValueError(f"{name} must have shape ({rows},), got {tuple(t.shape)}")
    return _as(t, dtype)


def _ptr(t: torch.Tensor | None) -> int:
    return t.data_ptr() if t is not None else 0


def _row_stride(t: torch.Tensor | None) -> int:
    return t.stride(0) if t is not None else 0


def apply_logit_rules(logits: torch.Tensor, rules: LogitRules, out: torch.Tensor | None = None) -> torch.Tensor:
    """``rules`` on logits (B, V), computed in fp32 and rounded once to the
    logits' dtype; into ``out`` (which may be ``logits``) or a new tensor."""
    dev = logits.get_device()
    tokens, bias_tokens, bias_values, allowed = rules.tokens, rules.bias_tokens, rules.bias_values, rules.allowed
    for t in rules.tensors():
        if t.get_device() != dev or dev < 0:
            _same_device(dev, logits, t)
    if dev < 0:
        _same_device(dev, logits)
    if dev != _current_device():
        with torch.cuda.device(dev):
            return apply_logit_rules(logits, rules, out)
    _no_grad(logits)
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
    width = None
    history = biases = 0
    if tokens is not None:
        width = tokens.dtype
        if width is not torch.int64 and width is not torch.int32:
            raise TypeError(f"tokens must be int32 or int64, got {width}")
        tokens = _rows_of(tokens, rows, "tokens")
        history = tokens.shape[1]
    elif not (rules.token_lens is rules.prompt_lens is rules.repetition_penalty is rules.presence_penalty
              is rules.frequency_penalty is None):
        raise ValueError("penalties and lengths need tokens")
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias_tokens and bias_values go together")
    if bias_tokens is not None:
        if bias_tokens.dtype is not torch.int64 and bias_tokens.dtype is not torch.int32:
            raise TypeError(f"bias_tokens must be int32 or int64, got {bias_tokens.dtype}")
        if bias_tokens.shape != bias_values.shape:
            raise ValueError("bias_tokens and bias_values must have one shape")
        bias_tokens = _rows_of(bias_tokens, rows, "bias_tokens")
        if width is not None and bias_tokens.dtype is not width:  # both as the wider: narrowing could alias ids
            tokens, bias_tokens = tokens.to(torch.int64), bias_tokens.to(torch.int64)
        width = bias_tokens.dtype
        if bias_values.dtype is not torch.float32:
            bias_values = bias_values.to(torch.float32)
        bias_values = _rows_of(bias_values, rows, "bias_values")
        biases = bias_tokens.shape[1]
    if allowed is not None:
        if allowed.dtype is not torch.int32 or allowed.dim() != 2 or allowed.shape[1] < (vocab + 31) // 32:
            raise ValueError(f"allowed must be int32 ({rows}, at least {(vocab + 31) // 32})")
        allowed = _rows_of(allowed, rows, "allowed")
    lens = _per_row(rules.token_lens, rows, torch.int32, "token_lens")
    prompt = _per_row(rules.prompt_lens, rows, torch.int32, "prompt_lens")
    rep = _per_row(rules.repetition_penalty, rows, torch.float32, "repetition_penalty")
    pres = _per_row(rules.presence_penalty, rows, torch.float32, "presence_penalty")
    freq = _per_row(rules.frequency_penalty, rows, torch.float32, "frequency_penalty")
    lib = _native.load()
    ws_bytes = lib.plora_logit_rules_workspace(rows, vocab, history, biases)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=logits.device) if ws_bytes else None
    args = _native.LOGIT_RULES_ARGS.pack(
        logits.data_ptr(), row if rows > 1 else vocab, out.data_ptr(), out.stride(0) if rows > 1 else vocab, rows, vocab,
        dtype_code(logits.dtype), _ptr(tokens), _row_stride(tokens), history, _ptr(lens), _ptr(prompt), _ptr(rep),
        _ptr(pres), _ptr(freq), _ptr(bias_tokens), _row_stride(bias_tokens), _ptr(bias_values),
        _row_stride(bias_values), biases, _ptr(allowed), _row_stride(allowed), 4 if width is torch.int32 else 8,
        _ptr(ws), ws_bytes,
    )
    status = lib.plora_logit_rules(args, _raw_stream(dev))
    if status:
        _native.check("plora_logit_rules", status)
    return out
