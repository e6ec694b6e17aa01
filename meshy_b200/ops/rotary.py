"""Rotary positions beyond a base alone: both layouts, part of a head, scaled for long contexts.

:func:`.functional.qkv_rope` turns whole heads in the half layout by angles ``p theta^(-2 i / hd)``. :class:`Rope`
describes the other forms that checkpoints come with, and :func:`qkv_rotary` applies them to a fused QKV projection,
with QK-norm before them where a model has it, and with their gradient:

* half (pairs ``(i, i + rot / 2)``) or interleaved layout (pairs ``(2 i, 2 i + 1)``);
* the first ``rotary_dim`` channels of a head turned, the rest left as they are;
* frequencies scaled for contexts longer than the model was trained on (:class:`RopeScaling`).

:func:`qkv_rotary_to_cache` writes K and V of a step into the paged cache as well. On CUDA each call is one native kernel
on the current stream (two for the gradient with QK-norm) and can be captured in a CUDA graph; on the CPU the functions
of :mod:`.reference` run. Angles are exact to 2^-32 of a turn at every int32 position.
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field, fields
from fractions import Fraction
from functools import lru_cache
from typing import Any, Mapping

import torch

from . import reference as ref
from ._ext import ext
from .checks import check_range
from .functional import native

#: 2 pi to 200 bits
_TWO_PI = Fraction(2 * 314159265358979323846264338327950288419716939937510582097494459, 10 ** 62)


@dataclass(frozen=True)
class RopeScaling:
    """How frequencies ``f`` are stretched over a longer context, under the names of HF's ``rope_scaling``.

    * ``linear``: ``f / factor``;
    * ``llama3``: ``f / factor`` for pairs that make fewer than ``low_freq_factor`` turns over the original context,
      ``f`` for those that make more than ``high_freq_factor``, linear in the turns between;
    * ``yarn``: the same between ``beta_slow`` and ``beta_fast`` turns, linear in the pair's index (whole indices with
      ``truncate``), and the turned channels multiplied by ``attention_factor`` (default ``0.1 ln(factor) + 1``).
    """

    rope_type: str
    factor: float
    original_max_position_embeddings: int = 0
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None
    truncate: bool = True

    def __post_init__(self):
        if self.rope_type not in ("linear", "llama3", "yarn"):
            raise ValueError(f"rope_scaling: rope_type must be 'linear', 'llama3' or 'yarn', got {self.rope_type!r}")
        if not (math.isfinite(self.factor) and self.factor >= 1.0):
            raise ValueError(f"rope_scaling: factor must be finite and at least 1, got {self.factor}")
        if self.rope_type != "linear" and not self.original_max_position_embeddings > 0:
            raise ValueError(f"rope_scaling: {self.rope_type} needs original_max_position_embeddings")
        if self.rope_type == "llama3" and not 0.0 < self.low_freq_factor < self.high_freq_factor < math.inf:
            raise ValueError("rope_scaling: low_freq_factor must be positive and below high_freq_factor")
        if self.rope_type == "yarn" and not 0.0 < self.beta_slow < self.beta_fast < math.inf:
            raise ValueError("rope_scaling: beta_slow must be positive and below beta_fast")
        if self.attention_factor is not None and not (math.isfinite(self.attention_factor) and self.attention_factor > 0):
            raise ValueError(f"rope_scaling: attention_factor must be positive, got {self.attention_factor}")

    @classmethod
    def of(cls, scaling: "RopeScaling | Mapping[str, Any] | None") -> "RopeScaling | None":
        """From a mapping with HF's keys (``type`` for ``rope_type`` too); ``None`` or type ``default``: no scaling."""
        if scaling is None or isinstance(scaling, cls):
            return scaling
        values = {k: v for k, v in scaling.items() if v is not None}
        if "type" in values:
            values.setdefault("rope_type", values.pop("type"))
            values.pop("type", None)
        if values.get("rope_type") == "default":
            return None
        names = {f.name for f in fields(cls)}
        if unknown := sorted(set(values) - names):
            raise ValueError(f"rope_scaling: unknown keys {unknown}")
        if missing := sorted({"rope_type", "factor"} - set(values)):
            raise ValueError(f"rope_scaling: missing keys {missing}")
        return cls(**values)


@dataclass(frozen=True)
class Rope:
    """Rotary positions of heads of ``head_dim`` channels, of which the first ``rotary_dim`` (default: all) are turned."""

    head_dim: int
    theta: float = 1e4
    rotary_dim: int | None = None
    interleaved: bool = False
    scaling: RopeScaling | Mapping[str, Any] | None = None
    #: what the turned channels are multiplied by
    factor: float = field(init=False, compare=False)
    _tables: dict = field(default_factory=dict, init=False, repr=False, compare=False)

    def __post_init__(self):
        rot = self.head_dim if self.rotary_dim is None else self.rotary_dim
        if self.head_dim <= 0 or self.head_dim > 256 or self.head_dim % 8:
            raise ValueError(f"rope: head_dim must be a multiple of 8, at most 256, got {self.head_dim}")
        if rot <= 0 or rot > self.head_dim or rot % 8:
            raise ValueError(f"rope: rotary_dim must be a multiple of 8, at most head_dim {self.head_dim}, got {rot}")
        if not (math.isfinite(self.theta) and self.theta > 1.0):
            raise ValueError(f"rope: theta must be finite and above 1, got {self.theta}")
        object.__setattr__(self, "rotary_dim", rot)
        s = RopeScaling.of(self.scaling)
        object.__setattr__(self, "scaling", s)
        yarn = s is not None and s.rope_type == "yarn"
        factor = (s.attention_factor or 0.1 * math.log(s.factor) + 1.0) if yarn else 1.0
        object.__setattr__(self, "factor", factor)

    def frequencies(self) -> list[float]:
        """Radians per position of each of the ``rotary_dim / 2`` pairs."""
        rot, s = self.rotary_dim, self.scaling
        f = [self.theta ** (-2 * i / rot) for i in range(rot // 2)]
        if s is None:
            return f
        if s.rope_type == "linear":
            return [x / s.factor for x in f]
        n = s.original_max_position_embeddings
        if s.rope_type == "llama3":
            turns = [n * x / (2 * math.pi) for x in f]
            keep = [(t - s.low_freq_factor) / (s.high_freq_factor - s.low_freq_factor) for t in turns]
        else:
            lo, hi = (rot * math.log(n / (t * 2 * math.pi)) / (2 * math.log(self.theta))
                      for t in (s.beta_fast, s.beta_slow))  # indices whose pairs make so many turns
            if s.truncate:
                lo, hi = math.floor(lo), math.ceil(hi)
            lo, hi = max(lo, 0), min(hi, rot - 1)
            keep = [1 - (i - lo) / max(hi - lo, 1e-3) for i in range(rot // 2)]
        return [x / s.factor + min(max(k, 0.0), 1.0) * (x - x / s.factor) for x, k in zip(f, keep)]

    def turns(self, device) -> torch.Tensor:
        """``[rotary_dim / 2]`` int64: turns per position times 2^64, modulo 2^64. Made once per device for all ropes that
        are equal."""
        t = self._tables.get(device)
        if t is None:
            if not isinstance(device, torch.device):
                return self.turns(torch.device(device))
            t = self._tables[device] = _turn_table(self, device)
        return t


@lru_cache(maxsize=None)  # kept for good: captured graphs read them, and one is half a kilobyte
def _turn_table(rope: Rope, device: torch.device) -> torch.Tensor:
    if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("rope: make one call on this device before a CUDA graph capture (it uploads a table)")
    words = []
    for f in rope.frequencies():
        n, d = f.as_integer_ratio()
        n, d = (n << 64) * _TWO_PI.denominator, d * _TWO_PI.numerator
        w = (2 * n + d) // (2 * d) % (1 << 64)
        words.append(w - (1 << 64) if w >> 63 else w)
    with torch.inference_mode(False):  # (a backward pass may save it)
        return torch.tensor(words, dtype=torch.int64, device=device)


@lru_cache(maxsize=256)
def make_rope(head_dim: int, theta: float, rotary_dim: int | None, interleaved: bool,
              scaling: RopeScaling | None) -> Rope:
    """One :class:`Rope` (and one table per device) for all that ask for the same."""
    return Rope(head_dim, theta, rotary_dim, interleaved, scaling)


def _check(qkv, positions, rope, n_heads, n_kv, q_norm, k_norm):
    if qkv.dim() != 2 or n_heads <= 0 or n_kv <= 0 or qkv.shape[1] != (n_heads + 2 * n_kv) * rope.head_dim:
        raise ValueError(f"rotary: qkv must be [rows, {(n_heads + 2 * n_kv) * rope.head_dim}], got {list(qkv.shape)}")
    if positions.dtype != torch.int32 or positions.shape != qkv.shape[:1]:
        raise ValueError(f"rotary: positions must be int32 [{qkv.shape[0]}], got {positions.dtype} {list(positions.shape)}")
    if (q_norm is None) != (k_norm is None):
        raise ValueError("rotary: both norm weights or none")


def qkv_rotary(qkv: torch.Tensor, positions: torch.Tensor, rope: Rope, n_heads: int, n_kv: int,
               q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6):
    """``q [T, Hq, hd], k, v [T, Hkv, hd]`` of ``qkv [T, (Hq + 2 Hkv) hd]`` at ``positions [T]`` (int32): the heads split,
    RMS-normed with ``q_norm`` / ``k_norm [hd]`` where given, and turned. In fp32 between reading and writing, rounded
    once. Differentiable in ``qkv`` and the norms' weights (into the ``main_grad`` that they have in the backward pass,
    if any), once and backward only; the weights' sums have a fixed order."""
    if native(qkv):
        return ext().qkv_rotary(qkv, positions, rope.turns(qkv.device), rope.factor, rope.interleaved, q_norm, k_norm,
                                n_heads, n_kv, rope.head_dim, eps)
    _check(qkv, positions, rope, n_heads, n_kv, q_norm, k_norm)
    return ref.qkv_rotary(qkv, positions, rope, n_heads, n_kv, q_norm, k_norm, eps)


def qkv_rotary_to_cache(qkv, positions, rope: Rope, n_heads: int, n_kv: int, q_norm, k_norm, eps, k_cache, v_cache,
                        slot_mapping, *, keep_kv: bool = False):
    """:func:`qkv_rotary` with K and V written into the paged caches ``[pages, Hkv, page, hd]`` at ``slot_mapping [T]``
    int64 (slots outside the cache are skipped), without gradient. Returns ``q`` and, with ``keep_kv``, ``k, v``."""
    check_range("KV-cache slots", slot_mapping, 0, k_cache.shape[0] * k_cache.shape[2], skip_negative=True)
    if native(qkv):
        return ext().rotary_fwd(qkv, positions, rope.turns(qkv.device), rope.factor, rope.interleaved, q_norm, k_norm,
                                n_heads, n_kv, rope.head_dim, float(eps), k_cache, v_cache, slot_mapping, keep_kv)
    from .decode import kv_write

    _check(qkv, positions, rope, n_heads, n_kv, q_norm, k_norm)
    q, k, v = ref.qkv_rotary(qkv, positions, rope, n_heads, n_kv, q_norm, k_norm, eps)
    ok = (slot_mapping >= 0) & (slot_mapping < k_cache.shape[0] * k_cache.shape[2])
    kv_write(k[ok], v[ok], k_cache, v_cache, slot_mapping[ok])
    return (q, k, v) if keep_kv else (q, None, None)


__all__ = ["Rope", "RopeScaling", "make_rope", "qkv_rotary", "qkv_rotary_to_cache"]
