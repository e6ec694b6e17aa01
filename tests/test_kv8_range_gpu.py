"""Attention over the 8-bit KV cache at the ends of the cache's range, against 64 bits: keys and values of up to 2^126, rows
that one CTA has and rows that are cut and joined."""

import math

import pytest
import torch

from test_kv8_gpu import _check, _exact, _filled, _q, _rows

pytestmark = pytest.mark.gpu

LENS = {128: [1, 16, 700, 33, 0], 64: [1, 40, 513, 0, 3]}


def _refill(c, bt, lens, k_power=0, v_power=0, top=None, seed=50):
    """The rows' tokens anew, K and V times powers of two; ``top``: that value in some channels."""
    from meshy_b200.ops.kv8 import kv8_write

    Hkv, page, hd = c.k.shape[1:]
    for i, n in enumerate(lens):
        if not n:
            continue
        t = torch.arange(n)
        slots = bt[i].cpu()[t // page].long() * page + t % page
        k, v = (_rows(n, Hkv, hd, seed + 2 * i + j).float().clamp(-3.9, 3.9) * 2.0 ** p
                for j, p in enumerate((k_power, v_power)))
        if top is not None:
            k[t % 5 == 0, :, 3] = top
            v[t % 7 == 0, :, 5] = -top
        kv8_write(k.bfloat16().cuda(), v.bfloat16().cuda(), c, slots.cuda())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("k_power, q_power, scale_power", [
    (124, -100, -24), (124, -124, 0), (124, 0, -124), (120, -60, -60), (110, 10, -120), (124, -40, -130), (116, -116, 0),
    (-90, 126, -36), (-90, 100, -10), (0, 126, -126)])
def test_large_keys(hd, k_power, q_power, scale_power):
    """Scores of ordinary size from far factors."""
    lens = LENS[hd]
    c, bt = _filled(lens, 2, hd, 16)
    _refill(c, bt, lens, k_power=k_power)
    q = (_q(5, 12, hd).float().clamp(-1.9, 1.9) * 2.0 ** q_power).bfloat16()
    assert bool(q.isfinite().all())
    got = _check(q, c, bt, lens, 2.0 ** scale_power)
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("v_power", [100, 116, 121, 123, 124])
@pytest.mark.parametrize("lens", [None, [20011], [3000] * 4])
def test_large_values(hd, v_power, lens):
    """Short rows, where one CTA has all and single tokens carry a head, and long ones, which are cut and joined."""
    lens = lens or LENS[hd]
    c, bt = _filled(lens, 2, hd, 64)
    _refill(c, bt, lens, v_power=v_power)
    for scale in (None, 2.0, 0.0):
        got = _check(_q(len(lens), 14, hd), c, bt, lens, scale)
        assert bool(got.isfinite().all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("top", [2.0 ** 126, math.inf, 3e38])
def test_what_the_cache_clamps(hd, top):
    """Infinities and what lies above 2^126 are kept as 2^126; tiny queries, and none at all, meet them."""
    lens = LENS[hd]
    c, bt = _filled(lens, 2, hd, 32)
    _refill(c, bt, lens, k_power=124, v_power=124, top=top)
    for q_power in (-125, -110):
        q = (_q(5, 12, hd).float().clamp(-1.9, 1.9) * 2.0 ** q_power).bfloat16()
        assert bool(_check(q, c, bt, lens, 2.0 ** (-126 - q_power)).isfinite().all())
    assert bool(_check(torch.zeros_like(q), c, bt, lens).isfinite().all())


@pytest.mark.parametrize("v_power", [0, 60, 118])
@pytest.mark.parametrize("peak", [0, 40000])
def test_a_long_tail_under_large_values(v_power, peak):
    """One key ahead of 65535 others by a factor 2^22, which have large values: their common weight, 2^-6, has to arrive."""
    from meshy_b200.ops.kv8 import kv8_empty, kv8_write

    L, hd = 65536, 128
    k = torch.zeros(L, 1, hd, device="cuda")
    k[peak, 0, 0] = 16.0
    v = torch.full((L, 1, hd), 10.0, device="cuda")
    v += (torch.arange(hd, device="cuda") % 2) * 2
    v[peak] = 100.0
    c = kv8_empty(L // 64, 1, 64, hd, "cuda")
    kv8_write(k.bfloat16(), (v * 2.0 ** v_power).bfloat16(), c, torch.arange(L, device="cuda"))
    q = torch.zeros(1, 2, hd, device="cuda").bfloat16()
    q[..., 0] = 1.0
    bt = torch.arange(L // 64, dtype=torch.int32, device="cuda")[None]
    got = _check(q, c, bt, [L], 22 * math.log(2) / 16)
    # and the tail alone would have been missed: it is far more than the check's bound
    want, size, _, _ = _exact(q, c, bt, [L], 22 * math.log(2) / 16)
    assert bool(((100.0 * 2.0 ** v_power - want).abs() > 2.0 ** -7 * size).all()) and bool(got.isfinite().all())
