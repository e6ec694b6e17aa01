"""Blocks of the 8-bit KV cache that fill up token by token: what the growths of the scale cost the earlier tokens (CPU)."""

import pytest
import torch

from meshy_b200.ops import kv8 as K


def rows(kind, H, hd, seed=0):
    """16 tokens, as bf16."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(16, H, hd, generator=g)
    t = torch.arange(16.0)[:, None, None]
    if kind != "gaussian":
        x = x / x.abs().amax((1, 2), keepdim=True)
    if kind == "rising":
        x = x * 1.02 ** t
    elif kind == "doubling":
        x = x * 2.0 ** t
    elif kind == "falling":
        x = x * 0.9 ** t
    elif kind == "mixed":
        x = x * 2.0 ** torch.randint(-6, 7, (16, 1, 1), generator=g)
    return x.bfloat16()


def fill(x, cache, order=range(16), write=K.kv8_write):
    """One token after the other into block 1, K and its negative as V; the scales [16, H] after each."""
    scales = []
    for t in order:
        write(x[t:t + 1], -x[t:t + 1], cache, torch.tensor([16 + t], device=cache.k.device))
        scales.append(cache.scale[1, :, 0, 0].double().cpu())
    return torch.stack(scales)


def bound(scales):
    """[16, H, 1]: half a step at a token's write, and half of the then step at every growth after it. fp32 adds its
    roundings of the scales (2^-24 of them) and, once more, of the values read (127 steps at most)."""
    grown = torch.cat([torch.ones_like(scales[:1], dtype=torch.bool), scales[1:] != scales[:-1]])
    own = torch.stack([scales[t] + (scales * grown)[t + 1:].sum(0) for t in range(16)])
    return (own / 2 * (1 + 2.0 ** -23) + scales[-1] * 127 * 2.0 ** -23)[..., None]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["gaussian", "rising", "doubling", "falling", "mixed"])
def test_errors_add_up_to_half_the_sum_of_the_scales(kind, hd):
    for seed in range(4):
        x, c = rows(kind, 3, hd, seed), K.kv8_empty(2, 3, 16, hd, "cpu")
        scales = fill(x, c)
        growths = (scales[1:] > scales[:-1]).sum(0)
        assert bool((scales[1:] >= scales[:-1]).all())  # (of each head; the rows are normed over all)
        k, v = K.kv8_read(c, torch.arange(16, 32), torch.float64)
        allowed = bound(scales)
        assert bool(((k - x.double()).abs() <= allowed).all()) and bool(((v + x.double()).abs() <= allowed).all())
        assert bool((allowed <= scales[-1][:, None] * ((1 + growths) / 2 + 2.0 ** -15)[:, None]).all())
        # the same tokens in one write: half a step
        one = K.kv8_empty(2, 3, 16, hd, "cpu")
        K.kv8_write(x, -x, one, torch.arange(16, 32))
        assert torch.equal(one.scale[1, :, 0, 0].double(), scales[-1])
        off = (K.kv8_read(one, torch.arange(16, 32), torch.float64)[0] - x.double()).abs()
        assert bool((off <= scales[-1][:, None] * (0.5 + 127 * 2.0 ** -23)).all())


def test_small_growths_keep_the_level_and_stretch_the_value():
    """Largest values (1 + t / 128) / 2, one unit of bf16 after the other: r goes from 254 to floor(254 / (1 + 15 / 128)) =
    227 by steps of 1 or 2, and level 50 times any of these quotients rounds to 50 again (50 * 2 / 227 < 1 / 2)."""
    hd = 64
    x = torch.zeros(16, 1, hd)
    x[:, 0, 0] = (1 + torch.arange(16) / 128) / 2
    x[0, 0, 1] = 50 / 254
    x, c = x.bfloat16(), K.kv8_empty(2, 1, 16, hd, "cpu")
    scales = fill(x, c)
    assert float(scales[0]) == float(torch.tensor(1 / 254)) and float(scales[-1]) == float(torch.tensor(1 / 227))
    assert int((scales[1:] != scales[:-1]).sum()) == 15 and int(c.k[1, 0, 0, 1]) == 128 + 50
    off = float(K.kv8_read(c, torch.tensor([16]), torch.float64)[0][0, 0, 1]) - float(x[0, 0, 1])
    step = 1 / 227
    # 50 (1 - 227 / 254) = 5.3 steps; the bf16 channel itself is within 2^-11 of 50 / 254
    assert abs(off / step - 50 * (1 - 227 / 254)) < 227 * 2.0 ** -11 + 1e-3
    assert off <= float(bound(scales)[0, 0, 0]) <= 8 * step * (1 + 1e-4)
