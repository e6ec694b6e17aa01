"""8-bit KV cache on the CPU: the format against its definition, appended tokens, the attention over it, refusals."""

import math

import pytest
import torch

from meshy_b200.ops import checks
from meshy_b200.ops import kv8 as K


def _steps(top: float) -> float:
    """The largest number of 8 significant bits that is not above 127 / top."""
    m, e = math.frexp(127.0 / min(max(top, 2.0 ** -100), 2.0 ** 126))
    return math.ldexp(math.floor(m * 256) / 256, e)


def _level(x: float, r: float) -> int:
    return round(min(max(x, -(2.0 ** 126)), 2.0 ** 126) * r)  # (halves to even)


def _rows(T, H, hd, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, H, hd, generator=g) * spread).bfloat16()


def test_bytes_and_scales_of_whole_blocks():
    T, H, hd = 37, 2, 64
    c = K.kv8_empty(4, H, 16, hd, "cpu")
    k, v = _rows(T, H, hd), _rows(T, H, hd, 1, 1e-3)
    slots = torch.arange(T) + 16
    ko, vo = K.kv8_write(k, v, c, slots, keep=True)
    for x, data, kv, out in ((k, c.k, 0, ko), (v, c.v, 1, vo)):
        for b in range(0, T, 16):
            for h in range(H):
                block = x[b:b + 16, h].double()
                r = _steps(float(block.abs().max()))
                a = float(torch.tensor(1.0 / r, dtype=torch.float32))
                assert float(c.scale[1 + b // 16, h, 0, kv]) == a
                for t in range(len(block)):
                    n = [_level(y, r) for y in block[t].tolist()]
                    assert data[1 + b // 16, h, t].tolist() == [y + 128 for y in n]
                    want = torch.tensor([a * y for y in n], dtype=torch.float64).float().bfloat16()
                    assert torch.equal(out[b + t, h], want)
    assert torch.equal(K.kv8_read(c, slots, torch.bfloat16)[0], ko)


def test_round_trip_within_half_a_step():
    for spread in (1e-30, 1.0, 1e30):
        x = _rows(160, 2, 128, 3, spread)
        c = K.kv8_empty(10, 2, 16, 128, "cpu")
        K.kv8_write(x, -x, c, torch.arange(160))
        k, v = K.kv8_read(c, torch.arange(160), torch.float64)
        # r has lost less than 2^-7 of 127 / max, the scale half a step of fp32, the value as much
        step = x.double().abs().view(10, 16, 2, 128).amax((1, 3)).repeat_interleave(16, 0)[..., None] / 127 * (1 + 2.0 ** -7)
        bound = step * (0.5 + 128 * 2.0 ** -23)
        assert bool(((k - x.double()).abs() <= bound).all()) and bool(((v + x.double()).abs() <= bound).all())


def test_appended_tokens_follow_the_definition():
    hd, page = 64, 32
    c = K.kv8_empty(3, 1, page, hd, "cpu")
    x = _rows(page, 1, hd, 5)
    x = (x.float() * 2.0 ** torch.tensor([0, 1, 0, 4, -3, 5, 5, 9] * 4)[:, None, None]).bfloat16()
    held = []  # n of the block's tokens
    r = math.inf
    for t in range(page):
        if t % 16 == 0:
            held, r = [], math.inf
        K.kv8_write(x[t:t + 1], x[t:t + 1], c, torch.tensor([page + t]))
        new = min(r, _steps(float(x[t].abs().max())))
        if new < r:
            held = [[round(n * new / r) for n in row] for row in held]  # 15 bits over 8: no quotient near a half is cut
        r = new
        held.append([_level(y, r) for y in x[t, 0].double().tolist()])
        at = t // 16 * 16
        assert (c.k[1, 0, at:at + len(held)].long() - 128).tolist() == held, t
        assert float(c.scale[1, 0, t // 16, 1]) == float(torch.tensor(1.0 / r, dtype=torch.float32))
    # the same token again changes nothing
    before = [y.clone() for y in c]
    K.kv8_write(x[-1:], x[-1:], c, torch.tensor([page + page - 1]))
    assert all(torch.equal(a, b) for a, b in zip(before, c))


def test_extremes_and_nan():
    c = K.kv8_empty(6, 1, 16, 64, "cpu")
    x = torch.zeros(5, 1, 64)
    x[1] = 2.0 ** -120
    x[2, 0, 0], x[2, 0, 1], x[2, 0, 2] = math.inf, -math.inf, 1.0
    x[3, 0, 9] = math.nan
    x[4, 0, ::2], x[4, 0, 1::2] = 1.0, -0.5
    K.kv8_write(x, x, c, torch.arange(5) * 16 + 16)
    k, _ = K.kv8_read(c, torch.arange(5) * 16 + 16, torch.float32)
    assert bool((k[0] == 0).all()) and bool((k[1] == 0).all())
    assert bool(k[2].isfinite().all()) and k[2, 0, 0] == -k[2, 0, 1] and 0.99 < float(k[2, 0, 0]) / 2.0 ** 126 < 1.01
    assert bool(k[3].isnan().all())
    assert float(k[4, 0, 0]) == 1.0 and float(k[4, 0, 1]) == pytest.approx(-64 / 127, abs=1e-6)  # 63.5: to even
    # a NaN stays until the block is begun anew
    K.kv8_write(x[4:], x[4:], c, torch.tensor([16 * 4 + 1]))
    assert bool(K.kv8_read(c, torch.tensor([16 * 4 + 1]))[0].isnan().all())
    K.kv8_write(x[4:], x[4:], c, torch.tensor([16 * 4]))
    assert float(K.kv8_read(c, torch.tensor([16 * 4]), torch.float32)[0][0, 0, 0]) == 1.0


def test_slots_outside_are_skipped():
    c = K.kv8_empty(2, 2, 16, 64, "cpu")
    x = _rows(4, 2, 64)
    slots = torch.tensor([-1, 3, 32, 1 << 40])
    k, v = K.kv8_write(x, x, c, slots, keep=True)
    assert bool((k[[0, 2, 3]] == 0).all()) and bool((k[1] != 0).any()) and torch.equal(k, v)
    assert int(((c.k != 0) & (c.k != 128)).any(-1).sum()) == 2  # one token of two heads (128: the rest of its block, zeros)


def test_attention_against_64_bits():
    g = torch.Generator().manual_seed(2)
    hd, page, H = 64, 16, 2
    c = K.kv8_empty(9, H, page, hd, "cpu")
    lens = [40, 0, 1, 33, 100]
    bt = torch.full((5, 4), -1, dtype=torch.int32)
    bt[0, :3], bt[2, :1], bt[3, :3] = torch.tensor([4, 1, 7]), 2, torch.tensor([3, 0, 8])
    bt[4] = torch.tensor([5, 100, -3, 6])  # pages outside the cache; a length past the table
    q = torch.randn(5, 6, hd, generator=g)
    k, v = torch.randn(9 * page, H, hd, generator=g), torch.randn(9 * page, H, hd, generator=g)
    K.kv8_write(k, v, c, torch.arange(9 * page))
    kk, vv = K.kv8_read(c, torch.arange(9 * page), torch.float64)
    out = K.paged_attention_kv8(q, c, bt, torch.tensor(lens, dtype=torch.int32))
    for b, n in enumerate(lens):
        t = torch.arange(min(n, 4 * page))
        pg = bt[b, t // page].long()
        there = (pg >= 0) & (pg < 9)
        at = (pg * page + t % page)[there]
        for h in range(6):
            if len(at) == 0:
                assert float(out[b, h].abs().sum()) == 0.0
                continue
            p = torch.softmax(kk[at, h // 3] @ q[b, h].double() / math.sqrt(hd), 0)
            assert torch.allclose(out[b, h].double(), p @ vv[at, h // 3], atol=1e-5)


def test_cache_over_bytes():
    n = 3 * 2 * (32 // 16) * K.block_bytes(128)
    raw = torch.zeros(n + 7, dtype=torch.uint8)
    c = K.kv8_from_bytes(raw, 3, 2, 32, 128)
    assert c.page_size == 32 and c.head_dim == 128 and sum(t.numel() * t.element_size() for t in c) == n
    K.kv8_write(_rows(5, 2, 128), _rows(5, 2, 128, 1), c, torch.arange(5) + 32)
    assert int((raw != 0).sum()) > 0
    with pytest.raises(ValueError, match="bytes needed"):
        K.kv8_from_bytes(raw[:n - 1], 3, 2, 32, 128)


@pytest.mark.parametrize("n_kv, page, hd", [(2, 16, 32), (2, 8, 64), (2, 0, 64), (0, 16, 64), (2, 24, 128)])
def test_geometry_that_the_kernels_do_not_take(n_kv, page, hd):
    with pytest.raises(ValueError):
        K.kv8_empty(2, n_kv, page, hd, "cpu")
    with pytest.raises(ValueError):
        K.kv8_from_bytes(torch.zeros(1 << 16, dtype=torch.uint8), 1, n_kv, page, hd)


def test_debug_mode_names_rows_of_a_block_that_stand_apart():
    c = K.kv8_empty(4, 1, 16, 64, "cpu")
    x = _rows(3, 1, 64)
    checks.set_enabled(True)
    try:
        with pytest.raises(IndexError, match="stand together"):
            K.kv8_write(x, x, c, torch.tensor([16, 33, 17]))
        with pytest.raises(IndexError, match="outside"):
            K.kv8_write(x, x, c, torch.tensor([16, 17, 64]))
        K.kv8_write(x, x, c, torch.tensor([17, 16, -1]))
    finally:
        checks.set_enabled(False)
