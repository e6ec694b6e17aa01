"""Block tables and slot maps of a paged KV cache, made from request lengths on their device (no autograd).

* :func:`assign_pages` -- newly allocated pages into the rows of a block table that need them;
* :func:`token_maps` -- positions, cache slots and packed offsets of the rows' new tokens (a prompt's, or one of a decode
  step), as the rotary embedding, the cache write and the attention take them.

On CUDA each is one native kernel on the current stream and can be captured in a CUDA graph: lengths and pages are read
on the device. On the CPU the functions of :mod:`.reference` run.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import reference as ref
from ._ext import ext
from .checks import check_range, enabled


class TokenMaps(NamedTuple):
    positions: torch.Tensor   # [total] int32
    slots: torch.Tensor       # [total] int64: page * page_size + offset, -1 where there is none
    cu_seqlens: torch.Tensor  # [n + 1] int32


def _check(block_table, vectors: dict) -> None:
    if block_table.dtype != torch.int32 or block_table.dim() != 2:
        raise ValueError(f"block_table must be int32 [rows, pages], got {block_table.dtype} {list(block_table.shape)}")
    n = None
    for name, t in vectors.items():
        if t.dtype != torch.int32 or t.dim() != 1 or (n is not None and t.shape[0] != n):
            raise ValueError(f"{name} must be int32 [{'rows' if n is None else n}], got {t.dtype} {list(t.shape)}")
        n = t.shape[0]


def assign_pages(block_table: torch.Tensor, rows: torch.Tensor, have: torch.Tensor, need: torch.Tensor,
                 pages: torch.Tensor) -> None:
    """Deal ``pages [P]`` out in order: row ``rows[i]`` of ``block_table [R, M]`` gets the next ``need[i] - have[i]`` (none
    below zero) at columns ``have[i], ..``. All int32; ``rows`` distinct. What falls outside the table is not written,
    pages that no row needs stay out, and columns that the pages do not reach keep what they hold."""
    if enabled():
        check_range("block-table rows", rows, 0, block_table.shape[0], skip_negative=True)
        check_range("block-table columns", need, 0, block_table.shape[1] + 1)
    if block_table.is_cuda:
        ext().assign_pages(block_table, rows, have, need, pages)
        return
    _check(block_table, {"rows": rows, "have": have, "need": need})
    if pages.dtype != torch.int32 or pages.dim() != 1:
        raise ValueError(f"pages must be int32 [P], got {pages.dtype} {list(pages.shape)}")
    ref.assign_pages(block_table, rows, have, need, pages)


def token_maps(block_table: torch.Tensor, rows: torch.Tensor, start: torch.Tensor, lens: torch.Tensor, total: int,
               page_size: int) -> TokenMaps:
    """Maps of the tokens ``start[i] .. start[i] + lens[i] - 1`` of each row ``rows[i]`` (int32; lengths below zero count as
    zero), packed row after row. ``total``: entries of the result, at least the lengths' sum unless the tokens behind are
    not wanted; entries behind the last token have position 0 and slot -1, which the cache writes skip. A token whose row
    or page lies outside the table, or whose page id is negative, has slot -1 too."""
    if enabled():
        check_range("block-table rows", rows, 0, block_table.shape[0], skip_negative=True)
    if block_table.is_cuda:
        return TokenMaps(*ext().token_maps(block_table, rows, start, lens, int(total), int(page_size)))
    _check(block_table, {"rows": rows, "start": start, "lens": lens})
    if total < 0 or page_size <= 0:
        raise ValueError(f"total must not be negative and page_size positive, got {total} and {page_size}")
    return TokenMaps(*ref.token_maps(block_table, rows, start, lens, int(total), int(page_size)))


__all__ = ["TokenMaps", "assign_pages", "token_maps"]
