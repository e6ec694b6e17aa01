"""Logit controls of a decode step: penalties for repeated tokens, biases and token masks (no autograd).

For a request whose prompt and output so far contain the set ``seen`` and whose output contains token ``v`` ``c[v]``
times, the controlled logits are::

    z'[v] = rep(z[v]) - frequency * c[v] - presence * [c[v] > 0] + bias[v],    -inf where the mask forbids v
    rep(z) = z / repetition if z > 0 else z * repetition     for v in seen, z elsewhere

(the penalties of SGLang's and OpenAI's sampling parameters of the same names). :class:`LogitControls` holds the
device state of a fixed number of request slots:

* :func:`load_tokens` -- token state of requests when they are admitted, from their tokens so far;
* :func:`apply_logit_controls` -- count the tokens sampled last, then control the logits; on fp32 logits in place,
  which touches only the entries that change.

On CUDA each function is one native kernel on the current stream and can be captured in a CUDA graph.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Mapping, Sequence

import torch

from . import reference as ref
from ._ext import ext
from .checks import check_range


_FP32 = torch.finfo(torch.float32)


def _words(vocab: int) -> int:
    return (vocab + 31) // 32


def token_bits(tokens: Sequence[int], vocab: int) -> torch.Tensor:
    """``[ceil(vocab / 32)]`` int32 bitmask (CPU) with the bits of ``tokens`` set: token ``v`` is bit ``v % 32`` of word
    ``v // 32``."""
    flags = torch.zeros(_words(vocab) * 32, dtype=torch.int64)
    ids = torch.as_tensor(list(tokens), dtype=torch.int64)
    if ids.numel() and (int(ids.min()) < 0 or int(ids.max()) >= vocab):
        raise ValueError(f"token ids must be in [0, {vocab})")
    flags[ids] = 1
    w = (flags.view(-1, 32) << torch.arange(32)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


@dataclass
class LogitControls:
    """Device state of ``R`` request slots over a vocabulary of ``V`` (``W = ceil(V / 32)`` words of bits a row)."""

    repetition: torch.Tensor  # [R] fp32, 1: off
    frequency: torch.Tensor   # [R] fp32, 0: off
    presence: torch.Tensor    # [R] fp32, 0: off
    seen: torch.Tensor        # [R, W] int32 bits: token in the prompt or the output (bits past V are ignored)
    counts: torch.Tensor      # [R, V] int32: times the token was generated; a token with a count is a seen one
    bias_ids: torch.Tensor    # [R, K] int32, -1: unused; distinct within a row
    bias_vals: torch.Tensor   # [R, K] fp32
    mask: torch.Tensor        # [R, W] int32 bits: token allowed
    mask_on: torch.Tensor     # [R] int32: the mask counts

    def __post_init__(self):
        self.state = [self.repetition, self.frequency, self.presence, self.seen, self.counts, self.bias_ids,
                      self.bias_vals, self.mask, self.mask_on]

    @classmethod
    def create(cls, slots: int, vocab: int, *, device, max_bias: int = 64) -> "LogitControls":
        """All slots empty and every control off."""
        if slots <= 0 or vocab <= 0 or max_bias < 0:
            raise ValueError("logit controls: slots and vocabulary must be positive, max_bias not negative")
        W = _words(vocab)
        i32 = dict(dtype=torch.int32, device=device)
        return cls(torch.ones(slots, device=device), torch.zeros(slots, device=device), torch.zeros(slots, device=device),
                   torch.zeros(slots, W, **i32), torch.zeros(slots, vocab, **i32),
                   torch.full((slots, max_bias), -1, **i32), torch.zeros(slots, max_bias, device=device),
                   torch.full((slots, W), -1, **i32), torch.zeros(slots, **i32))

    @property
    def vocab(self) -> int:
        return self.counts.shape[1]

    @property
    def max_bias(self) -> int:
        return self.bias_ids.shape[1]

    def set_slot(self, slot: int, *, repetition_penalty: float = 1.0, frequency_penalty: float = 0.0,
                 presence_penalty: float = 0.0, logit_bias: Mapping[int, float] | None = None,
                 allowed_tokens: Sequence[int] | None = None) -> None:
        """The controls of one slot (defaults: off). Its token state is :func:`load_tokens`'s."""
        self._check_slot(slot)
        if allowed_tokens is not None:
            allowed_tokens = [int(t) for t in allowed_tokens]
        check_controls(self.vocab, self.max_bias, repetition_penalty, frequency_penalty, presence_penalty, logit_bias,
                       allowed_tokens)
        self.repetition[slot] = float(repetition_penalty)
        self.frequency[slot] = float(frequency_penalty)
        self.presence[slot] = float(presence_penalty)
        self.bias_ids[slot] = -1
        if logit_bias:
            n = len(logit_bias)
            self.bias_ids[slot, :n] = torch.tensor([int(v) for v in logit_bias], dtype=torch.int32)
            self.bias_vals[slot, :n] = torch.tensor([float(x) for x in logit_bias.values()])
        self.set_mask(slot, None if allowed_tokens is None else token_bits(allowed_tokens, self.vocab))

    def _check_slot(self, slot: int) -> None:
        if not 0 <= slot < self.counts.shape[0]:
            raise ValueError(f"logit controls: slot {slot} outside [0, {self.counts.shape[0]})")

    def set_mask(self, slot: int, bits: torch.Tensor | None) -> None:
        """Token mask of one slot as a bitmask ``[W]`` int32 (see :func:`token_bits`); ``None``: every token allowed."""
        self._check_slot(slot)
        if bits is not None:
            if bits.dtype != torch.int32 or bits.shape != self.mask.shape[1:]:
                raise ValueError(f"token mask must be int32 [{self.mask.shape[1]}], got {bits.dtype} {list(bits.shape)}")
            self.mask[slot].copy_(bits)
        self.mask_on[slot] = 0 if bits is None else 1


def check_controls(vocab: int, max_bias: int, repetition_penalty: float = 1.0, frequency_penalty: float = 0.0,
                   presence_penalty: float = 0.0, logit_bias: Mapping[int, float] | None = None,
                   allowed_tokens: Sequence[int] | None = None) -> None:
    """``ValueError`` unless the values of one request are usable (they are held in fp32, where 1e39 is no number and
    1e-50 is zero)."""
    if not (_FP32.tiny <= repetition_penalty <= _FP32.max):
        raise ValueError(f"repetition_penalty must be positive, got {repetition_penalty}")
    for name, x in (("frequency_penalty", frequency_penalty), ("presence_penalty", presence_penalty)):
        if not abs(x) <= _FP32.max:
            raise ValueError(f"{name} must be finite, got {x}")
    if logit_bias:
        if len(logit_bias) > max_bias:
            raise ValueError(f"logit_bias has {len(logit_bias)} entries, at most {max_bias}")
        ids = [int(v) for v in logit_bias]
        if len(set(ids)) < len(ids) or min(ids) < 0 or max(ids) >= vocab:
            raise ValueError(f"logit_bias token ids must be distinct and in [0, {vocab})")
        if not all(abs(float(x)) <= _FP32.max for x in logit_bias.values()):
            raise ValueError("logit_bias values must be finite (allowed_tokens forbids tokens)")
    if allowed_tokens is not None:
        ids = [int(v) for v in allowed_tokens]
        if not ids or min(ids) < 0 or max(ids) >= vocab:
            raise ValueError(f"allowed_tokens must name at least one token, all in [0, {vocab})")


def load_tokens(ctl: LogitControls, slots: torch.Tensor, tokens: torch.Tensor, cu_tokens: torch.Tensor,
                n_prompt: torch.Tensor) -> None:
    """Rewrite the token state of ``slots [n]`` (int32 or int64, distinct; negative: skipped): row ``i``'s tokens are
    ``tokens[cu_tokens[i]:cu_tokens[i + 1]]``, the first ``n_prompt[i]`` of them its prompt. Token ids outside the
    vocabulary are ignored."""
    check_range("logit-control slots", slots, 0, ctl.counts.shape[0], skip_negative=True)
    if ctl.counts.is_cuda:
        ext().load_tokens(ctl.state, slots, tokens, cu_tokens, n_prompt)
        return
    ref.load_tokens(ctl, slots, tokens, cu_tokens, n_prompt)


def apply_logit_controls(logits: torch.Tensor, ctl: LogitControls, slots: torch.Tensor, *,
                         new_tokens: torch.Tensor | None = None, done: torch.Tensor | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """Controlled logits (fp32) of ``logits [B, V]`` (fp32 or bf16), row ``b`` under the controls of ``slots[b]``
    (int32 or int64; negative: none). ``new_tokens [B]`` int64: the token each row sampled last is first counted as
    generated (negative: none; ``done [B]`` int32 nonzero: not counted). Rows that count must have distinct slots.
    ``out``: fp32 result; by default fp32 logits are rewritten in place."""
    check_range("logit-control slots", slots, 0, ctl.counts.shape[0], skip_negative=True)
    if out is None:
        out = logits if logits.dtype == torch.float32 else torch.empty(logits.shape, dtype=torch.float32,
                                                                       device=logits.device)
    if logits.is_cuda:
        ext().apply_logit_controls(logits, ctl.state, slots, new_tokens, done, out)
        return out
    return ref.apply_logit_controls(logits, ctl, slots, new_tokens, done, out)


__all__ = ["LogitControls", "apply_logit_controls", "check_controls", "load_tokens", "token_bits"]
