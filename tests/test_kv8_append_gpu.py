"""Blocks of the 8-bit KV cache that fill up token by token, on the GPU: the bytes of the CPU's form, and its bound."""

import pytest
import torch

from meshy_b200.ops import kv8 as K
from test_kv8_append_cpu import bound, fill, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H", [1, 3, 8])
@pytest.mark.parametrize("kind", ["gaussian", "rising", "doubling", "falling", "mixed"])
def test_bytes_of_blocks_that_fill_up(kind, H, hd):
    for seed in range(3):
        x = rows(kind, H, hd, seed)
        cpu, gpu = K.kv8_empty(2, H, 16, hd, "cpu"), K.kv8_empty(2, H, 16, hd, "cuda")
        scales = fill(x, cpu)
        assert torch.equal(fill(x.cuda(), gpu), scales)
        assert all(torch.equal(a, b.cpu()) for a, b in zip(cpu, gpu))
        k, v = (y.double().cpu() for y in K.kv8_read(gpu, torch.arange(16, 32, device="cuda")))
        allowed = bound(scales) + x.double().abs() * 2.0 ** -8 + bound(scales) * 2.0 ** -8  # the values are read in bf16
        assert bool(((k - x.double()).abs() <= allowed).all()) and bool(((v + x.double()).abs() <= allowed).all())


def test_many_blocks_side_by_side():
    """A batch whose rows each append to a block of their own, as a decode step does, some blocks further than others."""
    B, H, hd = 40, 2, 128
    x = torch.stack([rows("mixed", H, hd, s) for s in range(B)], 1)  # [16, B, H, hd]
    cpu, gpu = K.kv8_empty(B + 1, H, 16, hd, "cpu"), K.kv8_empty(B + 1, H, 16, hd, "cuda")
    for t in range(16):
        on = torch.tensor([b for b in range(B) if t < 16 - b % 5])
        slots = (on + 1) * 16 + t
        K.kv8_write(x[t, on], -x[t, on], cpu, slots)
        K.kv8_write(x[t, on].cuda(), -x[t, on].cuda(), gpu, slots.cuda())
    assert all(torch.equal(a, b.cpu()) for a, b in zip(cpu, gpu))
