"""Refusals of the rotary embedding that writes into the paged cache (GPU; all raise on the host)."""

import pytest
import torch

from meshy_b200.ops.rotary import Rope, qkv_rotary_to_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_caches_off_the_boundary(which, offset):
    """A cache that begins inside 8 bytes: stores of 8 bytes would be misaligned."""
    T, Hq, Hkv, hd, pages, page = 3, 4, 2, 64, 2, 16
    n = pages * Hkv * page * hd
    raw = [torch.zeros(n + 8, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    at = [offset if i == which else 0 for i in range(2)]
    caches = [x[o:o + n].view(pages, Hkv, page, hd) for x, o in zip(raw, at)]
    qkv = torch.randn(T, (Hq + 2 * Hkv) * hd, device="cuda").bfloat16()
    pos, slots = torch.arange(T, dtype=torch.int32, device="cuda"), torch.arange(T, device="cuda")
    with pytest.raises(RuntimeError, match="8-byte boundaries"):
        qkv_rotary_to_cache(qkv, pos, Rope(hd), Hq, Hkv, None, None, 1e-6, *caches, slots)
    torch.cuda.synchronize()
    assert all(float(x.abs().sum()) == 0.0 for x in raw)
    # four elements on, it is on a boundary again
    caches = [x[o // offset * 4 if o else 0:][:n].view(pages, Hkv, page, hd) for x, o in zip(raw, at)]
    q, k, v = qkv_rotary_to_cache(qkv, pos, Rope(hd), Hq, Hkv, None, None, 1e-6, *caches, slots, keep_kv=True)
    assert torch.equal(caches[0][0, :, :T].transpose(0, 1), k) and torch.equal(caches[1][0, :, :T].transpose(0, 1), v)
