"""4-bit KV cache on the CPU: the format against its definition in 64 bits, the attention over it, and refusals."""

import math

import pytest
import torch

from meshy_b200.ops import kv4 as K


def _slots(n, pages, page, seed=0):
    return torch.randperm(pages * page, generator=torch.Generator().manual_seed(seed))[:n]


def _bound(x, hd):
    """Largest distance of a stored value from ``x``: half a step, and the fp16 roundings of scale and base."""
    g = x.double().clamp(-65504, 65504).unflatten(-1, (hd // 64, 64))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    step = (hi - lo) / 15
    # the rounded scale spans 15 a >= (hi - lo)(1 - 2^-11), the base moves by 2^-11 |lo|; 2^-24: fp16's subnormal grid
    return (0.5 * step * (1 + 2 ** -11) + (hi - lo) * 2 ** -11 + lo.abs() * 2 ** -11 + 16 * 2 ** -24).expand_as(g).flatten(-2)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("spread", [1e-6, 1.0, 300.0])
def test_round_trip_within_half_a_step(hd, spread):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(37, 3, hd, generator=g) * spread + 2 * spread * torch.randn(1, 3, hd, generator=g)).bfloat16()
    c = K.kv4_empty(4, 3, 16, hd, "cpu")
    slots = _slots(37, 4, 16)
    K.kv4_write(x, -x, c, slots)
    k, v = K.kv4_read(c, slots, torch.float64)
    assert bool(((k - x.double()).abs() <= _bound(x, hd)).all())
    assert bool(((v + x.double()).abs() <= _bound(-x, hd)).all())


def test_word_layout():
    """Channel 64 g + 8 u + e is nibble e of word u G + g."""
    hd = 128
    x = torch.zeros(1, 1, hd)
    x[0, 0, :64] = torch.arange(64) % 16
    x[0, 0, 64:] = 15 - torch.arange(64) % 16
    c = K.kv4_empty(1, 1, 16, hd, "cpu")
    K.kv4_write(x, x, c, torch.tensor([3]))
    nib = torch.stack([c.k[0, 0, 3] & 15, c.k[0, 0, 3] >> 4], -1).reshape(-1).long()
    for ch in (0, 1, 9, 63, 64, 77, 127):
        grp, u, e = ch // 64, ch % 64 // 8, ch % 8
        assert int(nib[(u * 2 + grp) * 8 + e]) == int(x[0, 0, ch])
    assert c.scale[0, 0, 3, 0].tolist() == [[1.0, 0.0], [1.0, 0.0]]


def test_constant_extreme_and_nan_groups():
    x = torch.zeros(4, 1, 128)
    x[1] = 7.5                # a = 0: the base alone
    x[2, 0, :64] = torch.linspace(-1e38, 1e38, 64)  # beyond fp16: clamped
    x[3, 0, 70] = float("nan")
    c = K.kv4_empty(1, 1, 16, 128, "cpu")
    K.kv4_write(x, x, c, torch.arange(4))
    k, _ = K.kv4_read(c, torch.arange(4), torch.float32)
    assert bool((k[0] == 0).all()) and bool((k[1] == 7.5).all())
    assert bool(k[2].isfinite().all()) and float(k[2, 0, 0]) == -65504.0
    assert bool(k[3, 0, 64:].isnan().all()) and bool((k[3, 0, :64] == 0).all())


@pytest.mark.parametrize("side", [70000.0, -70000.0, 3e38, -3e38, math.inf, -math.inf])
def test_groups_beyond_the_range_are_clamped(side):
    x = torch.zeros(1, 1, 128)
    x[..., :64] = side * (1 + torch.arange(64) % 3 / 16.0)
    c = K.kv4_empty(1, 1, 16, 128, "cpu")
    K.kv4_write(x, -x, c, torch.tensor([2]))
    k, v = K.kv4_read(c, torch.tensor([2]), torch.float32)
    assert torch.equal(k, x.clamp(-65504, 65504)) and torch.equal(v, -k)


def test_slots_outside_the_cache_are_skipped():
    c = K.kv4_empty(2, 1, 16, 64, "cpu")
    x = torch.ones(3, 1, 64)
    K.kv4_write(x, x, c, torch.tensor([-1, 5, 32]))
    k, _ = K.kv4_read(c, torch.tensor([5, -1, 40]), torch.float32)
    assert k[:, 0, 0].tolist() == [1.0, 0.0, 0.0] and int((c.scale != 0).sum()) == 2


def test_attention_matches_softmax_over_stored_values():
    g = torch.Generator().manual_seed(2)
    lens = [0, 1, 16, 33]
    c = K.kv4_empty(9, 2, 16, 64, "cpu")
    bt = torch.zeros(4, 3, dtype=torch.int32)
    order = torch.randperm(9, generator=g).int()
    at = 0
    for i, n in enumerate(lens):
        np_ = -(-n // 16)
        bt[i, :np_] = order[at:at + np_]
        at += np_
    every = torch.arange(9 * 16)
    K.kv4_write(torch.randn(144, 2, 64, generator=g), torch.randn(144, 2, 64, generator=g), c, every)
    q = torch.randn(4, 6, 64, generator=g)
    out = K.paged_attention_kv4(q, c, bt, torch.tensor(lens, dtype=torch.int32))
    k, v = K.kv4_read(c, every, torch.float64)
    assert bool((out[0] == 0).all())
    for i, n in enumerate(lens):
        rows = [int(bt[i, t // 16]) * 16 + t % 16 for t in range(n)]
        for h in range(6):
            if n:
                p = torch.softmax(k[rows, h // 3] @ q[i, h].double() / math.sqrt(64), 0)
                assert torch.allclose(out[i, h].double(), p @ v[rows, h // 3], rtol=1e-5, atol=1e-5)


def test_pages_and_lengths_outside_are_masked():
    g = torch.Generator().manual_seed(5)
    c = K.kv4_empty(4, 2, 16, 64, "cpu")
    K.kv4_write(torch.randn(64, 2, 64, generator=g), torch.randn(64, 2, 64, generator=g), c, torch.arange(64))
    q = torch.randn(1, 4, 64, generator=g)
    run = lambda pages, n: K.paged_attention_kv4(q, c, torch.tensor([pages], dtype=torch.int32), torch.tensor([n], dtype=torch.int32))
    want = run([2, 0], 32)
    assert torch.allclose(run([2, 0, 4, -1], 60), want) and torch.allclose(run([2, -7, 0], 48), want)
    assert torch.equal(run([2, 0], 1 << 30), want)
    assert bool((run([-1, 9], 20) == 0).all()) and bool((run([2, 0], -3) == 0).all())


def test_cache_over_bytes():
    assert K.row_bytes(128) == 144 and K.row_bytes(64) == 72
    raw = torch.zeros(3 * 2 * 16 * 144, dtype=torch.uint8)
    c = K.kv4_from_bytes(raw, 3, 2, 16, 128)
    K.kv4_write(torch.ones(1, 2, 128), torch.ones(1, 2, 128), c, torch.tensor([20]))
    assert c.page_size == 16 and c.head_dim == 128 and int((raw != 0).sum()) > 0
    with pytest.raises(ValueError, match="bytes needed"):
        K.kv4_from_bytes(raw[:-1], 3, 2, 16, 128)


@pytest.mark.parametrize("page,hd", [(16, 96), (24, 64), (0, 128)])
def test_unsupported_shapes_are_refused(page, hd):
    with pytest.raises(ValueError):
        K.kv4_empty(1, 1, page, hd, "cpu")


@pytest.mark.parametrize("n_kv,page,hd", [(1, 16, 32), (1, 16, 192), (2, 24, 64), (1, 0, 128), (0, 16, 64)])
def test_unsupported_shapes_are_refused_over_bytes_too(n_kv, page, hd):
    with pytest.raises(ValueError, match="4-bit KV cache"):
        K.kv4_from_bytes(torch.zeros(1 << 16, dtype=torch.uint8), 1, n_kv, page, hd)
    with pytest.raises(ValueError, match="4-bit KV cache"):
        K.kv4_empty(1, n_kv, page, hd, "cpu")
