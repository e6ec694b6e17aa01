"""Rows without a slot (below zero) are not written to the paged cache, whichever call writes it (CPU)."""

import pytest
import torch

from meshy_b200.ops import checks
from meshy_b200.ops import decode as D
from meshy_b200.ops.rotary import Rope


@pytest.mark.parametrize("checked", [False, True])
@pytest.mark.parametrize("rope", [None, Rope(64, rotary_dim=32)])
def test_a_row_without_a_slot_is_not_written(rope, checked):
    torch.manual_seed(0)
    T, Hq, Hkv, hd, pages, page = 6, 4, 2, 64, 3, 16
    qkv = torch.randn(T, (Hq + 2 * Hkv) * hd)
    pos = torch.arange(T, dtype=torch.int32)
    slots = torch.tensor([47, -1, 0, -17, 20, -1])
    caches = [torch.full((pages, Hkv, page, hd), 7.0) for _ in range(2)]
    checks.set_enabled(checked)
    try:
        q, k, v = D.qkv_rope_to_cache(qkv, pos, None, None, Hq, Hkv, hd, 1e4, 1e-6, *caches, slots, keep_kv=True, rope=rope)
        again = [torch.full_like(c, 7.0) for c in caches]
        D.kv_write(k, v, *again, slots)
    finally:
        checks.set_enabled(False)
    for x, cache, other in zip((k, v), caches, again):
        want = torch.full_like(cache, 7.0)
        for t in (0, 2, 4):
            want[slots[t] // page, :, slots[t] % page] = x[t]
        assert torch.equal(cache, want) and torch.equal(other, want)
