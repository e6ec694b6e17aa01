"""Paged KV cache in 4 bits: quantising write, read-back and decode attention (no autograd).

A row (one head of one token, ``hd`` = 64 or 128 channels) is kept in groups of 64 channels. A group holds a nibble
``n`` per channel and, in fp16, a scale ``a = (max - min) / 15`` and a base ``z = min``; a nibble stands for
``a n + z``. A token takes ``hd + hd / 8`` bytes per KV head for K and V together, against ``4 hd`` in bf16, so a
cache of the same size holds 3.55 times as many tokens.

* :func:`kv4_write` -- quantise this step's K/V rows into the cache (decode rows or a whole prompt);
* :func:`kv4_read` -- the values the cache holds at given slots (a prompt's attention reads its own K/V through it,
  so that prefill and decode see the same keys and values);
* :func:`paged_attention_kv4` -- decode attention over each row's pages.

On CUDA every function is one native kernel on the current stream and can be captured in a CUDA graph; slots and
pages outside the cache are skipped, so padding rows may carry -1. On the CPU the functions of
:mod:`.reference` run. Values are clamped to +-65504 (the range of fp16); a group with a NaN reads back as NaN.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import reference as ref
from ._ext import ext
from .checks import check_paged, check_range

GROUP = ref.KV4_GROUP


class KV4Cache(NamedTuple):
    """One layer's cache: ``k``, ``v`` ``[pages, Hkv, page, hd / 2]`` uint8 and ``scale [pages, Hkv, page, 2, hd / 64,
    2]`` fp16 (K and V, groups, (a, z)). 32-bit word ``w`` of a row holds channels ``64 (w mod G) + 8 (w div G) + 0..7``
    (``G = hd / 64``), lowest channel in the lowest nibble."""

    k: torch.Tensor
    v: torch.Tensor
    scale: torch.Tensor

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return 2 * self.k.shape[3]


def row_bytes(hd: int) -> int:
    """Bytes of the cache per token and KV head (K and V, nibbles and fp16 pairs)."""
    return hd + 8 * (hd // GROUP)


def check_geometry(n_kv: int, page: int, hd: int) -> None:
    """``ValueError`` for a cache that the kernels do not take."""
    if hd not in (64, 128):
        raise ValueError(f"4-bit KV cache: head_dim must be 64 or 128, got {hd}")
    if page <= 0 or page % 16:
        raise ValueError(f"4-bit KV cache: page size must be a multiple of 16, got {page}")
    if n_kv <= 0:
        raise ValueError(f"4-bit KV cache: at least one KV head is needed, got {n_kv}")


def kv4_empty(n_pages: int, n_kv: int, page: int, hd: int, device) -> KV4Cache:
    """A zeroed cache."""
    check_geometry(n_kv, page, hd)
    return KV4Cache(torch.zeros(n_pages, n_kv, page, hd // 2, dtype=torch.uint8, device=device),
                    torch.zeros(n_pages, n_kv, page, hd // 2, dtype=torch.uint8, device=device),
                    torch.zeros(n_pages, n_kv, page, 2, hd // GROUP, 2, dtype=torch.float16, device=device))


def kv4_from_bytes(raw: torch.Tensor, n_pages: int, n_kv: int, page: int, hd: int) -> KV4Cache:
    """A cache laid over ``raw`` (uint8, at least ``n_pages * n_kv * page * row_bytes(hd)`` of them, 16-byte aligned)."""
    check_geometry(n_kv, page, hd)
    n = n_pages * n_kv * page
    half = n * (hd // 2)
    if raw.dtype != torch.uint8 or raw.dim() != 1 or raw.numel() < n * row_bytes(hd):
        raise ValueError(f"4-bit KV cache: {n * row_bytes(hd)} bytes needed")
    return KV4Cache(raw[:half].view(n_pages, n_kv, page, hd // 2), raw[half:2 * half].view(n_pages, n_kv, page, hd // 2),
                    raw[2 * half:n * row_bytes(hd)].view(torch.float16).view(n_pages, n_kv, page, 2, hd // GROUP, 2))


def kv4_write(k: torch.Tensor, v: torch.Tensor, cache: KV4Cache, slot_mapping: torch.Tensor) -> None:
    """``k/v [T, Hkv, hd]`` (any strides) into ``cache`` at ``slot_mapping [T]`` int64; slots must be distinct."""
    check_range("KV-cache slots", slot_mapping, 0, cache.k.shape[0] * cache.k.shape[2], skip_negative=True)
    if k.is_cuda:
        ext().kv4_write(k, v, cache.k, cache.v, cache.scale, slot_mapping)
        return
    ref.kv4_write(k, v, cache, slot_mapping)


def kv4_read(cache: KV4Cache, slot_mapping: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """``k, v [T, Hkv, hd]``: the values the cache stands for at ``slot_mapping`` (zeros for a slot outside it)."""
    check_range("KV-cache slots", slot_mapping, 0, cache.k.shape[0] * cache.k.shape[2], skip_negative=True)
    if cache.k.is_cuda:
        if dtype != torch.bfloat16:
            raise ValueError(f"kv4_read: bfloat16 on CUDA, got {dtype}")
        return ext().kv4_read(cache.k, cache.v, cache.scale, slot_mapping)
    return ref.kv4_read(cache, slot_mapping, dtype)


def paged_attention_kv4(q: torch.Tensor, cache: KV4Cache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                        scale: float | None = None) -> torch.Tensor:
    """Decode attention of ``q [B, Hq, hd]`` over each row's first ``seq_lens [B]`` cached tokens, on the pages
    ``block_table [B, max_pages]``; query heads share the KV heads evenly. A row of length 0 gives zeros.

    Calls on one stream share a workspace, which the first call of a size on that stream allocates: make one before
    a capture on the stream, and replay graphs that were captured on one stream one after another."""
    check_paged("paged attention", block_table, seq_lens, cache.k.shape[0], cache.k.shape[2])
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    if q.is_cuda:
        return ext().kv4_attention(q, cache.k, cache.v, cache.scale, block_table, seq_lens, float(scale))
    return ref.attention_decode_kv4(q, cache, block_table, seq_lens, scale)


__all__ = ["KV4Cache", "check_geometry", "kv4_empty", "kv4_from_bytes", "kv4_read", "kv4_write", "paged_attention_kv4", "row_bytes"]
