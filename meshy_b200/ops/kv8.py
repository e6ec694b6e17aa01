"""Paged KV cache in 8 bits: quantising write, read-back and decode attention (no autograd).

The 16 tokens of a block (slots ``16 i .. 16 i + 15``) share one scale per head, K and V apart. With ``r`` the largest
number of 8 significant bits that is not above ``127 / max|x|``, a channel is kept as the byte ``rint(x r) + 128`` and the
scale as ``a = fp32(1 / r)``: byte ``u`` stands for ``a (u - 128)``. A token takes ``2 hd`` bytes and half a byte of scales per
KV head, against ``4 hd`` in bf16, so a cache of the same size holds 1.99 times as many tokens.

Blocks fill up in order. A write that holds a block's first token starts the block anew; any other keeps the smaller of
the block's ``r`` and its own, and where that shrinks it the block's other tokens are requantised, ``rint(n r' / r)``.

A channel written with its whole block is off by half a step ``a`` at most. In a block that fills up over several writes each
write that enlarges the scale rounds the earlier tokens once more, by half of its step. These add up: a token is off by at most
half the sum of the scales its block has had since it was written, ``(1 + g) / 2`` steps of the present one after ``g``
enlargements, and 8 after the 15 that a block filled token by token can have. (Where ``r'`` is only little below ``r`` the
level stays as it is and the value grows with the scale.) Gaussian rows appended one by one are off by 2.1 steps at most (root
mean square 0.36, in one write 0.29), rows that grow by 2 % each by 5.2 (1.5). So a sequence whose tokens are written anew in
one call reads other values than it decoded with.

* :func:`kv8_write` -- quantise this step's K/V rows into the cache (decode rows or whole prompts), and hand back the
  values now held (a prompt's attention reads its own K/V through them, so that prefill and decode see the same);
* :func:`kv8_read` -- the values the cache holds at given slots;
* :func:`paged_attention_kv8` -- decode attention over each row's pages.

On CUDA every function is one native kernel on the current stream and can be captured in a CUDA graph; slots and pages
outside the cache are skipped, so padding rows may carry -1. On the CPU the functions of :mod:`.reference` run. Values are
clamped to +-2^126; a block with a NaN reads back as NaN.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import reference as ref
from ._ext import ext
from .checks import check_paged, check_range, enabled

BLOCK = ref.KV8_BLOCK


class KV8Cache(NamedTuple):
    """One layer's cache: ``k``, ``v`` ``[pages, Hkv, page, hd]`` uint8 and ``scale [pages, Hkv, page / 16, 2]`` fp32 (K, V)."""

    k: torch.Tensor
    v: torch.Tensor
    scale: torch.Tensor

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]


def block_bytes(hd: int) -> int:
    """Bytes of the cache per block of 16 tokens and KV head (K and V, and their scales)."""
    return BLOCK * 2 * hd + 8


def check_geometry(n_kv: int, page: int, hd: int) -> None:
    """``ValueError`` for a cache that the kernels do not take."""
    if hd not in (64, 128):
        raise ValueError(f"8-bit KV cache: head_dim must be 64 or 128, got {hd}")
    if page <= 0 or page % BLOCK:
        raise ValueError(f"8-bit KV cache: page size must be a multiple of 16, got {page}")
    if n_kv <= 0:
        raise ValueError(f"8-bit KV cache: at least one KV head is needed, got {n_kv}")


def kv8_empty(n_pages: int, n_kv: int, page: int, hd: int, device) -> KV8Cache:
    """A zeroed cache."""
    check_geometry(n_kv, page, hd)
    u8 = dict(dtype=torch.uint8, device=device)
    return KV8Cache(torch.zeros(n_pages, n_kv, page, hd, **u8), torch.zeros(n_pages, n_kv, page, hd, **u8),
                    torch.zeros(n_pages, n_kv, page // BLOCK, 2, dtype=torch.float32, device=device))


def kv8_from_bytes(raw: torch.Tensor, n_pages: int, n_kv: int, page: int, hd: int) -> KV8Cache:
    """A cache laid over ``raw`` (uint8, at least ``n_pages * n_kv * page / 16 * block_bytes(hd)`` of them, 16-byte
    aligned)."""
    check_geometry(n_kv, page, hd)
    n = n_pages * n_kv * page
    size, half = n // BLOCK * block_bytes(hd), n * hd
    if raw.dtype != torch.uint8 or raw.dim() != 1 or raw.numel() < size:
        raise ValueError(f"8-bit KV cache: {size} bytes needed")
    return KV8Cache(raw[:half].view(n_pages, n_kv, page, hd), raw[half:2 * half].view(n_pages, n_kv, page, hd),
                    raw[2 * half:size].view(torch.float32).view(n_pages, n_kv, page // BLOCK, 2))


def _check_runs(slots: torch.Tensor, page: int) -> None:
    """Debug mode: rows of one block stand together and name each slot once (but for page 0, where idle rows write)."""
    if not enabled() or slots.numel() == 0:
        return
    b = torch.where(slots >= page, slots // BLOCK, -1)
    begins = b >= 0  # a run: the first row, and each whose block is not that of the row before (a skipped row has none)
    begins[1:] &= b[1:] != b[:-1]
    held = slots[b >= 0]
    if int(begins.sum()) != b[b >= 0].unique().numel():
        raise IndexError("kv8_write: rows whose slots lie in one block must stand together")
    if held.unique().numel() != held.numel():
        raise IndexError("kv8_write: a slot is given twice")


def kv8_write(k: torch.Tensor, v: torch.Tensor, cache: KV8Cache, slot_mapping: torch.Tensor, *, keep: bool = False):
    """``k/v [T, Hkv, hd]`` (any strides) into ``cache`` at ``slot_mapping [T]`` int64: distinct slots, those of one block on
    neighbouring rows in any order, with no other row between them, skipped ones included. What a block holds whose rows
    stand apart, or one of whose slots is given twice, is undefined: rows' pieces and scales may be mixed, its other tokens' too
    (only idle rows, on a page that nothing reads, may do so; other blocks are not touched). With ``keep``, the values that
    the cache now holds for these rows, ``(k', v')`` (zeros for a slot outside it)."""
    check_range("KV-cache slots", slot_mapping, 0, cache.k.shape[0] * cache.k.shape[2], skip_negative=True)
    _check_runs(slot_mapping, cache.k.shape[2])
    if k.is_cuda:
        return ext().kv8_write(k, v, cache.k, cache.v, cache.scale, slot_mapping, bool(keep))
    ref.kv8_write(k, v, cache, slot_mapping)
    return ref.kv8_read(cache, slot_mapping, k.dtype) if keep else None


def kv8_read(cache: KV8Cache, slot_mapping: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """``k, v [T, Hkv, hd]``: the values the cache stands for at ``slot_mapping`` (zeros for a slot outside it)."""
    check_range("KV-cache slots", slot_mapping, 0, cache.k.shape[0] * cache.k.shape[2], skip_negative=True)
    if cache.k.is_cuda:
        if dtype != torch.bfloat16:
            raise ValueError(f"kv8_read: bfloat16 on CUDA, got {dtype}")
        return ext().kv8_read(cache.k, cache.v, cache.scale, slot_mapping)
    return ref.kv8_read(cache, slot_mapping, dtype)


def paged_attention_kv8(q: torch.Tensor, cache: KV8Cache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                        scale: float | None = None) -> torch.Tensor:
    """Decode attention of ``q [B, Hq, hd]`` over each row's first ``seq_lens [B]`` cached tokens, on the pages
    ``block_table [B, max_pages]``; query heads share the KV heads evenly. A row of length 0 gives zeros."""
    check_paged("paged attention", block_table, seq_lens, cache.k.shape[0], cache.k.shape[2])
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    if q.is_cuda:
        return ext().kv8_attention(q, cache.k, cache.v, cache.scale, block_table, seq_lens, float(scale))
    return ref.attention_decode_kv8(q, cache, block_table, seq_lens, scale)


__all__ = ["KV8Cache", "block_bytes", "check_geometry", "kv8_empty", "kv8_from_bytes", "kv8_read", "kv8_write",
           "paged_attention_kv8"]
