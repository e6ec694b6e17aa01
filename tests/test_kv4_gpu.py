"""4-bit KV cache kernels against a plain implementation in 64 bits.

The write is compared bit for bit: every step of the format is an exactly rounded operation. The attention's result is
a bf16 number (relative rounding 2^-9) of a sum whose weights may be held in 11 bits or more and whose scores carry
fp32 sums: a weight's relative error is below 2^-11 (its rounding and that of its score, |score error| < 2^-12 for the
score sizes used here), so the numerator moves by at most 2^-11 max|v| and the normaliser by the same; with the
rounding that bounds the error by 2^-9 |o| + 2^-9 max|v|, max over the row's values.
"""

import math

import pytest
import torch

from meshy_b200.ops import kv4 as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def _value64(c, rows, kv):
    """Values ``[n, Hkv, hd]`` (fp64) of cache rows ``rows`` (page * page_size + offset), from the format's text."""
    data = (c.k, c.v)[kv]
    page, hd = c.page_size, c.head_dim
    G = hd // 64
    ch = torch.arange(hd, device=DEV)
    nib_at = ((ch % 64) // 8 * G + ch // 64) * 8 + ch % 8
    b = data[rows // page, :, rows % page].long()[..., nib_at // 2]
    n = (b >> (4 * (nib_at % 2))) & 15
    az = c.scale[rows // page, :, rows % page, kv].double()
    return az[..., ch // 64, 0] * n + az[..., ch // 64, 1]


def _expect(q, c, bt, lens, scale=None):
    """fp64 attention and the bound's max|v| per row and KV head."""
    B, Hq, hd = q.shape
    Hkv, page = c.k.shape[1], c.page_size
    rep = Hq // Hkv
    scale = 1 / math.sqrt(hd) if scale is None else scale
    out = torch.zeros(B, Hq, hd, dtype=torch.float64, device=DEV)
    vmax = torch.zeros(B, Hq, 1, dtype=torch.float64, device=DEV)
    for b, L in enumerate(lens):
        if L <= 0:
            continue
        t = torch.arange(L, device=DEV)
        rows = bt[b, t // page].long() * page + t % page
        k, v = _value64(c, rows, 0), _value64(c, rows, 1)
        p = torch.softmax(torch.einsum("grd,lgd->grl", q[b].double().view(Hkv, rep, hd), k) * scale, -1)
        out[b] = torch.einsum("grl,lgd->grd", p, v).reshape(Hq, hd)
        vmax[b] = v.abs().amax((0, 2)).repeat_interleave(rep)[:, None]
    return out, vmax


def _check(out, want, vmax):
    err = (out.double() - want).abs()
    assert bool((err <= 2 ** -9 * want.abs() + 2 ** -9 * vmax).all()), f"largest error {float(err.max())}"


def _setup(lens, Hq, Hkv, hd, page, seed=0, kscale=1.0, vscale=1.0, koff=0.0, extra_pages=2):
    """Cache with shuffled pages; the tail of every last page, the spare pages and unused table entries are
    poisoned (NaN scales, page ids outside the cache)."""
    g = _gen(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + extra_pages
    c = K.kv4_empty(P, Hkv, page, hd, DEV)
    c.k.random_(generator=g)
    c.v.random_(generator=g)
    c.scale.fill_(float("nan"))
    bt = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32, device=DEV)
    order = torch.randperm(P, generator=g, device=DEV)
    at = 0
    for i, n in enumerate(lens):
        pg = order[at:at + need[i]]
        at += need[i]
        bt[i, :need[i]] = pg.int()
        if n:
            t = torch.arange(n, device=DEV)
            k = kscale * (torch.randn(n, Hkv, hd, generator=g, device=DEV) + koff * torch.randn(1, Hkv, hd, generator=g, device=DEV))
            v = vscale * torch.randn(n, Hkv, hd, generator=g, device=DEV)
            K.kv4_write(k.bfloat16(), v.bfloat16(), c, pg[t // page] * page + t % page)
    q = torch.randn(len(lens), Hq, hd, generator=g, device=DEV).bfloat16()
    return q, c, bt, torch.tensor(lens, dtype=torch.int32, device=DEV)


# ── write and read-back ──────────────────────────────────────────────────────

@pytest.mark.parametrize("T,Hkv,hd,page", [(1, 1, 64, 16), (7, 2, 128, 64), (64, 2, 128, 64), (333, 8, 128, 48),
                                           (1000, 3, 64, 32), (13200, 5, 128, 64), (33000, 2, 64, 16), (70000, 1, 64, 64)])
@pytest.mark.parametrize("spread", [1e-6, 1.0, 1000.0])
def test_write_is_bit_exact(T, Hkv, hd, page, spread):
    from meshy_b200.ops import reference as ref

    g = _gen(T)
    slab = (torch.randn(T, 2 * Hkv, hd, generator=g, device=DEV) * spread
            + 3 * spread * torch.randn(1, 2 * Hkv, hd, generator=g, device=DEV)).bfloat16()
    k, v = slab[:, :Hkv], slab[:, Hkv:]  # strided, as the fused projection leaves them
    pages = -(-T // page) + 1
    c = K.kv4_empty(pages, Hkv, page, hd, DEV)
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:T]
    K.kv4_write(k, v, c, slots)
    for x, data, kv in ((k, c.k, 0), (v, c.v, 1)):
        b, pairs = ref.kv4_quantize(x.cpu())
        assert torch.equal(data[slots // page, :, slots % page].cpu(), b)
        assert torch.equal(c.scale[slots // page, :, slots % page, kv].cpu(), pairs)
    rk, rv = K.kv4_read(c, slots)
    assert torch.equal(rk, _value64(c, slots, 0).float().bfloat16())
    assert torch.equal(rv, _value64(c, slots, 1).float().bfloat16())
    unused = torch.ones(pages * page, dtype=torch.bool, device=DEV)
    unused[slots] = False
    rest = unused.nonzero().flatten()
    assert int(c.k[rest // page, :, rest % page].sum()) == 0 and int((c.scale[rest // page, :, rest % page] != 0).sum()) == 0


def test_write_special_values_and_ties():
    x = torch.zeros(8, 1, 128, device=DEV)
    x[1] = -7.5
    x[2, 0, :64] = torch.linspace(-1e38, 1e38, 64, device=DEV)
    x[3, 0, 5], x[3, 0, 70] = float("nan"), float("inf")
    x[4, 0, ::2] = -0.0
    x[5] = (torch.arange(128, device=DEV) % 31).float() / 2  # quotients on and between the halves
    x[6] = 1e-30 * torch.arange(128, device=DEV)             # below fp16: scale 0
    x[7, 0, 0] = 5e-8 * 15                                   # subnormal scale
    x = x.bfloat16()
    from meshy_b200.ops import reference as ref

    c = K.kv4_empty(1, 1, 16, 128, DEV)
    K.kv4_write(x, x, c, torch.arange(8, device=DEV))
    b, pairs = ref.kv4_quantize(x.cpu())
    assert torch.equal(c.k[0, 0, :8].cpu(), b[:, 0])
    got, want = c.scale[0, 0, :8, 0].cpu(), pairs[:, 0]
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_write_groups_beyond_the_range():
    """All channels of a group on one side of fp16's range: both extremes are clamped."""
    from meshy_b200.ops import reference as ref

    inf = float("inf")
    sides = [70000.0, -70000.0, 1e6, -1e6, 3e38, -3e38, inf, -inf, 65504.0, -65504.0]
    x = torch.zeros(2 * len(sides), 1, 128, device=DEV)
    for i, s in enumerate(sides):
        x[2 * i, 0, :64] = s                                            # constant
        x[2 * i + 1, 0, 64:] = s * (1 + torch.arange(64, device=DEV) % 3 / 16.0)  # spread, on the same side
    x = x.bfloat16()
    c = K.kv4_empty(2, 1, 16, 128, DEV)
    slots = torch.arange(len(x), device=DEV)
    K.kv4_write(x, -x, c, slots)
    for y, data, kv in ((x, c.k, 0), (-x, c.v, 1)):
        b, pairs = ref.kv4_quantize(y.cpu())
        assert torch.equal(data.transpose(1, 2).reshape(32, 1, 64)[slots].cpu(), b)
        assert torch.equal(c.scale.transpose(1, 2).reshape(32, 1, 2, 2, 2)[slots][:, :, kv].cpu(), pairs)
    k, v = K.kv4_read(c, slots)
    assert bool(k.isfinite().all()) and torch.equal(k, x.clamp(-65504, 65504)) and torch.equal(v, -k)


def test_every_scale_is_written_as_divided():
    """Each fp16 scale that a group can have, with channels at and around the halves: the quotients by multiplication
    have the bits of a division."""
    from meshy_b200.ops import reference as ref

    a = torch.arange(1, 0x7C00, dtype=torch.int16).view(torch.float16).float()
    a = a[15 * a <= 2 * 65504]
    span = (15 * a).to(DEV)
    hi = (span.view(torch.int32) & -65536).view(torch.float32)  # the upper 8 bits; the rest is a bf16 number too
    hi = torch.minimum(hi, torch.full_like(hi, 65280.0))
    lo = -(span - hi)
    g = _gen(11)
    x = lo[:, None] + span[:, None] * torch.rand(len(a), 64, generator=g, device=DEV)
    x[:, 32:] = lo[:, None] + a.to(DEV)[:, None] * (torch.randint(30, (len(a), 32), generator=g, device=DEV) / 2.0)
    x[:, 0], x[:, 63] = lo, hi
    x = x.bfloat16().clamp(lo.bfloat16()[:, None], hi.bfloat16()[:, None])[:, None]
    pages = -(-len(a) // 64)
    c = K.kv4_empty(pages, 1, 64, 64, DEV)
    slots = torch.arange(len(a), device=DEV)
    K.kv4_write(x, x, c, slots)
    b, pairs = ref.kv4_quantize(x.cpu())
    assert torch.equal(c.k.view(-1, 1, 32)[slots].cpu(), b)
    assert torch.equal(c.scale.view(-1, 1, 2, 1, 2)[slots][:, :, 0].cpu(), pairs)
    assert len(pairs[..., 0].unique()) > 0.9 * len(a)


def test_slots_outside_are_skipped_and_empty_calls():
    c = K.kv4_empty(2, 2, 16, 128, DEV)
    x = torch.ones(4, 2, 128, device=DEV).bfloat16()
    K.kv4_write(x, x, c, torch.tensor([-1, 5, 32, -(1 << 40)], device=DEV))
    k, v = K.kv4_read(c, torch.tensor([5, -1, 32, 1 << 40], device=DEV))
    assert k[:, 0, 0].tolist() == [1, 0, 0, 0] and v[:, 1, 127].tolist() == [1, 0, 0, 0]
    assert int((c.scale != 0).sum()) == 2 * 2 * 2
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    K.kv4_write(x[:0], x[:0], c, none)
    assert K.kv4_read(c, none)[0].shape == (0, 2, 128)


@pytest.mark.parametrize("make", [lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),
                                  lambda x: torch.cat([x.new_zeros(*x.shape[:2], 1), x], -1)[..., 1:],  # odd start
                                  lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),
                                  lambda x: torch.cat([x, x], -1)[..., :x.shape[-1]]])
def test_any_strides(make):
    g = _gen(3)
    x = torch.randn(21, 4, 128, generator=g, device=DEV).bfloat16()
    y = torch.randn(21, 4, 128, generator=g, device=DEV).bfloat16()
    slots = torch.randperm(48, generator=g, device=DEV)[:21]
    a, b = K.kv4_empty(3, 4, 16, 128, DEV), K.kv4_empty(3, 4, 16, 128, DEV)
    K.kv4_write(x, y, a, slots)
    K.kv4_write(make(x), make(y), b, slots)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(a.scale, b.scale)
    q = torch.randn(1, 8, 128, generator=g, device=DEV).bfloat16()
    bt = torch.arange(3, dtype=torch.int32, device=DEV)[None]
    n = torch.tensor([48], dtype=torch.int32, device=DEV)
    wide = torch.full((1, 9), -1, dtype=torch.int32, device=DEV)
    wide[:, 2:5] = bt
    assert torch.equal(K.paged_attention_kv4(q, a, bt, n), K.paged_attention_kv4(make(q), b, wide[:, 2:5], n))


# ── attention ────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("Hq,Hkv,hd", [(12, 2, 128), (14, 2, 64), (16, 2, 128), (32, 8, 128), (28, 4, 128), (4, 4, 64),
                                       (24, 2, 128), (17, 1, 128), (5, 5, 128)])
@pytest.mark.parametrize("page", [16, 64, 48])
def test_attention_heads_and_pages(Hq, Hkv, hd, page):
    lens = [0, 1, 2, 15, 16, 17, page - 1, page, page + 1, 127, 128, 129, 300, 1001]
    q, c, bt, n = _setup(lens, Hq, Hkv, hd, page, seed=Hq + hd)
    out = K.paged_attention_kv4(q, c, bt, n)
    want, vmax = _expect(q, c, bt, lens)
    _check(out, want, vmax)
    assert bool((out[0] == 0).all())


@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [65], [4097], [20000, 3], [70001], [1] * 300, [200] * 150 + [0, 9000]])
@pytest.mark.parametrize("Hq,Hkv,hd", [(12, 2, 128), (14, 2, 64)])
def test_attention_lengths(lens, Hq, Hkv, hd):
    q, c, bt, n = _setup(lens, Hq, Hkv, hd, 64, seed=len(lens))
    out = K.paged_attention_kv4(q, c, bt, n)
    _check(out, *_expect(q, c, bt, lens))
    assert torch.equal(out, K.paged_attention_kv4(q, c, bt, n))  # the same sums in the same order


@pytest.mark.parametrize("B,longest,page", [(2, 9000, 64), (5, 3000, 64), (37, 700, 16), (75, 2000, 64), (90, 400, 32),
                                            (149, 50, 64), (390, 90, 64), (800, 40, 48)])
@pytest.mark.parametrize("Hq,Hkv,hd", [(6, 1, 128), (16, 4, 64)])
def test_attention_ragged_splits(B, longest, page, Hq, Hkv, hd):
    """The work's cuts fall anywhere: between rows, inside them, behind a row's last token."""
    g = torch.Generator().manual_seed(B + longest)
    lens = (torch.rand(B, generator=g) ** 2 * (longest + 1)).long()
    lens[torch.randint(B, (max(1, B // 8),), generator=g)] = 0
    lens[int(torch.randint(B, (1,), generator=g))] = longest
    lens = lens.tolist()
    q, c, bt, n = _setup(lens, Hq, Hkv, hd, page, seed=B)
    out = K.paged_attention_kv4(q, c, bt, n)
    _check(out, *_expect(q, c, bt, lens))
    for b in (0, B // 2, B - 1):  # a row by itself: other cuts, the same numbers to rounding
        _check(K.paged_attention_kv4(q[b:b + 1], c, bt[b:b + 1], n[b:b + 1]), *_expect(q[b:b + 1], c, bt[b:b + 1], [lens[b]]))


def _count_setup(lens, Hq, Hkv, hd, page, seed, channel):
    """Keys of zero, so that every token has the same weight, and values that are one in channel ``channel(t, head)``
    (where that is one) and zero elsewhere: out[ch] is the number of a row's tokens with that channel, over its length."""
    g = _gen(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + 1
    c = K.kv4_empty(P, Hkv, page, hd, DEV)
    c.scale.fill_(float("nan"))
    bt = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32, device=DEV)
    order = torch.randperm(P, generator=g, device=DEV)
    want = torch.zeros(len(lens), Hkv, hd, dtype=torch.float64, device=DEV)
    one = 15 * float(torch.tensor(1 / 15).half())  # what the cache holds for 1
    at = 0
    for i, n in enumerate(lens):
        pg = order[at:at + need[i]]
        at += need[i]
        bt[i, :need[i]] = pg.int()
        if n:
            t = torch.arange(n, device=DEV)
            ch = channel(t[:, None], torch.arange(Hkv, device=DEV)[None])
            v = ((ch[..., None] == torch.arange(hd, device=DEV))).bfloat16()
            K.kv4_write(torch.zeros_like(v), v, c, pg[t // page] * page + t % page)
            want[i] = v.double().sum(0) * one / n
    q = torch.randn(len(lens), Hq, hd, generator=g, device=DEV).bfloat16()
    return q, c, bt, torch.tensor(lens, dtype=torch.int32, device=DEV), want.repeat_interleave(Hq // Hkv, 1)


def _check_counts(lens, Hq, Hkv, hd, page, seed, channel):
    # products of weights and scales are rounded to 11 bits (2^-11), the result to 8 (2^-8); a channel whose count is below
    # 200 shows one token more or less
    q, c, bt, n, want = _count_setup(lens, Hq, Hkv, hd, page, seed, channel)
    err = (K.paged_attention_kv4(q, c, bt, n).double() - want).abs()
    assert bool((err <= (2 ** -8 + 2 ** -10) * want).all()), float((err / want.clamp(min=1e-9)).max())


@pytest.mark.parametrize("Hq,Hkv,hd", [(12, 2, 128), (14, 2, 64), (17, 1, 128)])
@pytest.mark.parametrize("lens,page", [([1], 64), ([31, 32, 33, 63, 64, 65], 32), ([700], 64), ([3001, 0, 129, 1, 4097], 16),
                                       ([9000, 5, 8999], 48), ([20011], 64), ([70001], 32), ([257] * 150 + [3000], 64),
                                       ([100, 0, 7] * 100, 16), ([4096] * 8, 64), ([16384, 16383], 64)])
def test_no_block_of_tokens_is_lost_or_doubled(lens, page, Hq, Hkv, hd):
    for block in (1, 16, 32, 100):
        _check_counts(lens, Hq, Hkv, hd, page, len(lens) + block, lambda t, h: (t // block + h) % hd)


@pytest.mark.parametrize("lens,page,Hq,Hkv,hd", [([20011], 64, 8, 8, 128), ([9000], 48, 16, 4, 64), ([2500, 0, 5001, 77], 16, 8, 8, 64),
                                                 ([1500] * 20 + [33], 64, 16, 8, 128), ([70001], 64, 16, 16, 128)])
def test_every_token_counts_once(lens, page, Hq, Hkv, hd):
    """A window of hd tokens to a head, a token to a channel: wherever the work is cut, out[ch] is 1 / length."""
    for first in range(0, max(lens), hd * Hkv):
        _check_counts(lens, Hq, Hkv, hd, page, first, lambda t, h: t - first - h * hd)


@pytest.mark.parametrize("kscale,vscale,koff", [(1.0, 1e-4, 0.0), (1.0, 2000.0, 0.0), (4.0, 1.0, 0.0), (0.3, 1.0, 8.0),
                                                (1e-4, 1.0, 0.0), (0.0, 1.0, 0.0), (1.0, 0.0, 0.0)])
def test_attention_scales(kscale, vscale, koff):
    lens = [700, 3000]
    q, c, bt, n = _setup(lens, 12, 2, 128, 64, seed=5, kscale=kscale, vscale=vscale, koff=koff)
    _check(K.paged_attention_kv4(q, c, bt, n), *_expect(q, c, bt, lens))


@pytest.mark.parametrize("qscale", [1e-30, 1e-6, 200.0])
def test_attention_query_scales(qscale):
    lens = [900, 64]
    q, c, bt, n = _setup(lens, 12, 2, 128, 64, seed=6, kscale=1.0 / max(qscale, 1.0))
    q = (q.float() * qscale).bfloat16()
    for scale in (None, 0.25 / max(1.0, qscale) * 1.7):
        _check(K.paged_attention_kv4(q, c, bt, n, scale), *_expect(q, c, bt, lens, scale))


@pytest.mark.parametrize("peak", [0, 40000, 65535])
def test_attention_long_tail_keeps_its_mass(peak):
    """One key ahead of 65535 others by a factor 2^22: their common weight, 2^-6, has to arrive."""
    L, hd = 65536, 128
    k = torch.zeros(L, 1, hd, device=DEV)
    k[peak, 0, 0] = 16.0
    v = torch.full((L, 1, hd), 10.0, device=DEV)
    v += (torch.arange(hd, device=DEV) % 2) * 2
    v[peak] = 0
    c = K.kv4_empty(L // 64, 1, 64, hd, DEV)
    K.kv4_write(k.bfloat16(), v.bfloat16(), c, torch.arange(L, device=DEV))
    q = torch.zeros(1, 2, hd, device=DEV)
    q[..., 0] = 1.0
    scale = 22 * math.log(2) / 16
    bt = torch.arange(L // 64, dtype=torch.int32, device=DEV)[None]
    out = K.paged_attention_kv4(q.bfloat16(), c, bt, torch.tensor([L], dtype=torch.int32, device=DEV), scale)
    want, _ = _expect(q.bfloat16(), c, bt, [L], scale)
    assert bool(((out.double() - want).abs() <= 2 ** -7 * want.abs()).all())


@pytest.mark.parametrize("L", [700, 20000])
@pytest.mark.parametrize("every", [0, 100000, 256, 32])
def test_small_values_beside_tokens_of_large_ones(L, every):
    """Values that carry the result keep their precision beside tokens of next to no weight whose values spread a hundred
    thousand times as far, and below peaks that have no spread at all. Weights and their products with the scales are
    held in 11 bits, scores to 2^-12, the result in bf16: 2^-8 |o| + 2^-9 sum p |v|."""
    hd = 128
    g = _gen(12)
    t = torch.arange(L, device=DEV)
    k = torch.zeros(L, 1, hd, device=DEV)
    v = 10 + 4 * torch.rand(L, 1, hd, generator=g, device=DEV)
    k[t % 256 == 5, 0, 0] = 16.0         # a factor 2^22 ahead of the others
    v[t % 256 == 5] = 0
    if every:
        k[t % every == 0, 0, 0] = -64.0  # 2^-88 of the others
        v[t % every == 0] = 65504.0 * (torch.arange(hd, device=DEV) % 2 * 2 - 1)
    q = torch.zeros(1, 2, hd, device=DEV).bfloat16()
    q[..., 0] = 1.0
    scale = 22 * math.log(2) / 16
    bt = torch.arange(-(-L // 64), dtype=torch.int32, device=DEV)[None]
    c = K.kv4_empty(bt.shape[1], 1, 64, hd, DEV)
    K.kv4_write(k.bfloat16(), v.bfloat16(), c, t)
    out = K.paged_attention_kv4(q, c, bt, torch.tensor([L], dtype=torch.int32, device=DEV), scale)
    kk, vv = _value64(c, t, 0)[:, 0], _value64(c, t, 1)[:, 0]
    p = torch.softmax(kk @ q[0, 0].double() * scale, 0)
    want, size = p @ vv, (p * vv.abs().amax(1)).sum()
    err = (out[0].double() - want).abs()
    assert bool((err <= 2 ** -8 * want.abs() + 2 ** -9 * size).all()), float((err / size).max())


def test_attention_rising_scores():
    """Every tile's maximum above the last: the running maximum moves at every step, late keys carry the weight."""
    L, hd = 5000, 128
    k = torch.zeros(L, 2, hd, device=DEV)
    k[:, :, 0] = torch.arange(L, device=DEV)[:, None] * (60.0 / L)
    v = torch.randn(L, 2, hd, generator=_gen(1), device=DEV)
    c = K.kv4_empty(-(-L // 16), 2, 16, hd, DEV)
    K.kv4_write(k.bfloat16(), v.bfloat16(), c, torch.arange(L, device=DEV))
    bt = torch.arange(-(-L // 16), dtype=torch.int32, device=DEV)[None]
    n = torch.tensor([L], dtype=torch.int32, device=DEV)
    for sign in (1.0, -1.0):
        q = torch.zeros(1, 4, hd, device=DEV)
        q[..., 0] = sign * 8
        _check(K.paged_attention_kv4(q.bfloat16(), c, bt, n), *_expect(q.bfloat16(), c, bt, [L]))


def test_attention_nan_key_reaches_its_row_only():
    lens = [300, 300]
    q, c, bt, n = _setup(lens, 12, 2, 128, 64)
    slot = int(bt[0, 2]) * 64 + 7
    bad = torch.full((1, 2, 128), float("nan"), device=DEV).bfloat16()
    K.kv4_write(bad, torch.zeros_like(bad), c, torch.tensor([slot], device=DEV))
    out = K.paged_attention_kv4(q, c, bt, n)
    assert bool(out[0].isnan().all())
    want, vmax = _expect(q[1:], c, bt[1:], lens[1:])
    _check(out[1:], want, vmax)


def test_pages_and_lengths_outside_are_masked():
    q, c, bt, n = _setup([200], 12, 2, 128, 64)
    short, _ = _expect(q, c, bt, [128])
    bt2 = bt.clone()
    bt2[0, 2:] = c.k.shape[0] + 5  # the last pages are missing
    out = K.paged_attention_kv4(q, c, bt2, n)
    assert bool(((out.double() - short).abs() <= 2 ** -6).all())
    # a length beyond the table counts the table's pages; a negative one counts as 0
    full = K.paged_attention_kv4(q, c, bt[:, :2], torch.tensor([1 << 30], dtype=torch.int32, device=DEV))
    assert bool(((full.double() - short).abs() <= 2 ** -6).all())
    assert bool((K.paged_attention_kv4(q, c, bt, torch.tensor([-3], dtype=torch.int32, device=DEV)) == 0).all())


def test_length_at_the_end_of_32_bits():
    """A table that spans 2^31 tokens and a length of 2^31 - 1: rounding it up to whole units must not wrap."""
    q, c, bt, n = _setup([200], 2, 1, 128, 64)
    wide = torch.full((1, (1 << 25) + 1), -1, dtype=torch.int32, device=DEV)
    wide[:, :2] = bt[:, :2]
    n.fill_(2 ** 31 - 1)
    _check(K.paged_attention_kv4(q, c, wide, n), *_expect(q, c, bt, [128]))


def test_offsets_beyond_32_bits():
    page, Hkv, hd = 64, 2, 128
    P = (1 << 31) // (Hkv * page * hd // 2) + 64  # more than 2^31 bytes of K
    c = K.KV4Cache(torch.empty(P, Hkv, page, hd // 2, dtype=torch.uint8, device=DEV),
                   torch.empty(P, Hkv, page, hd // 2, dtype=torch.uint8, device=DEV),
                   torch.empty(P, Hkv, page, 2, 2, 2, dtype=torch.float16, device=DEV))
    g = _gen(9)
    pages = torch.tensor([P - 1, 0, P - 40], device=DEV)
    t = torch.arange(150, device=DEV)
    x = torch.randn(150, Hkv, hd, generator=g, device=DEV).bfloat16()
    K.kv4_write(x, -x, c, pages[t // page] * page + t % page)
    k, v = K.kv4_read(c, pages[t // page] * page + t % page)
    assert float((k.float() - x.float()).abs().max()) < 0.5 and torch.equal(k[:, :, 0].isfinite(), v[:, :, 0].isfinite())
    q = torch.randn(1, 12, hd, generator=g, device=DEV).bfloat16()
    bt = pages.int()[None]
    _check(K.paged_attention_kv4(q, c, bt, torch.tensor([150], dtype=torch.int32, device=DEV)), *_expect(q, c, bt, [150]))


def test_other_stream_and_graph():
    lens = [900, 40, 0, 5000]
    q, c, bt, n = _setup(lens, 12, 2, 128, 64)
    want = K.paged_attention_kv4(q, c, bt, n)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = K.paged_attention_kv4(q, c, bt, n)
    s.synchronize()
    assert torch.equal(want, other)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = K.paged_attention_kv4(q, c, bt, n)
    n.copy_(torch.tensor([3, 5000, 1, 900], dtype=torch.int32))  # lengths change between replays
    bt2 = bt[[0, 3, 1, 0]].clone()
    bt.copy_(bt2)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, K.paged_attention_kv4(q, c, bt, n))
    _check(out, *_expect(q, c, bt, [3, 5000, 1, 900]))


def test_two_streams_at_once():
    a = _setup([20000, 500], 12, 2, 128, 64, seed=1)
    b = _setup([7000] * 3, 14, 2, 64, 64, seed=2)
    wa, wb = K.paged_attention_kv4(*a), K.paged_attention_kv4(*b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            oa = K.paged_attention_kv4(*a)
        with torch.cuda.stream(s2):
            ob = K.paged_attention_kv4(*b)
        outs.append((oa, ob))
    torch.cuda.synchronize()
    assert all(torch.equal(oa, wa) and torch.equal(ob, wb) for oa, ob in outs)


def test_workspace_grows_with_the_segments():
    """More segments than the first counters hold (16384), on a stream that has used the smaller ones."""
    B, Hkv, hd, page = 2100, 8, 64, 16
    s = torch.cuda.Stream()
    small = _setup([40, 3000], 8, Hkv, hd, page, seed=3)
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 40, (B,), generator=g).tolist()
    many = _setup(lens, 8, Hkv, hd, page, seed=4)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        a = K.paged_attention_kv4(*small)
        b = [K.paged_attention_kv4(*many) for _ in range(2)]
        a2 = K.paged_attention_kv4(*small)
    s.synchronize()
    _check(a, *_expect(*small[:3], [40, 3000]))
    _check(b[0], *_expect(*many[:3], lens))
    assert torch.equal(a, a2) and torch.equal(*b)


def test_refusals():
    q, c, bt, n = _setup([100], 12, 2, 128, 64)
    k = torch.zeros(3, 2, 128, device=DEV).bfloat16()
    slots = torch.arange(3, device=DEV)
    bad = [lambda: K.kv4_write(k.float(), k, c, slots), lambda: K.kv4_write(k, k[:2], c, slots),
           lambda: K.kv4_write(k, k, c, slots.int()), lambda: K.kv4_write(k[:, :1], k[:, :1], c, slots),
           lambda: K.kv4_write(k[..., :64], k[..., :64], c, slots), lambda: K.kv4_write(k, k, c, slots.cpu()),
           lambda: K.kv4_write(k, k, c._replace(scale=c.scale.float()), slots),
           lambda: K.kv4_write(k, k, c._replace(k=c.k[:, :, ::2]), slots), lambda: K.kv4_read(c, slots, torch.float16),
           lambda: K.paged_attention_kv4(q.half(), c, bt, n), lambda: K.paged_attention_kv4(q[:, :3], c, bt, n),
           lambda: K.paged_attention_kv4(q, c, bt.long(), n), lambda: K.paged_attention_kv4(q, c, bt, n.long()),
           lambda: K.paged_attention_kv4(q, c, bt, n[:0]), lambda: K.paged_attention_kv4(q, c, bt.cpu(), n),
           lambda: K.paged_attention_kv4(q[..., :64], c, bt, n)]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            pytest.fail(f"call {i} was accepted")
    assert K.paged_attention_kv4(q[:0], c, bt[:0], n[:0]).shape == (0, 12, 128)


def test_a_cache_without_heads_is_refused():
    none = K.KV4Cache(torch.empty(2, 0, 16, 64, dtype=torch.uint8, device=DEV),
                      torch.empty(2, 0, 16, 64, dtype=torch.uint8, device=DEV),
                      torch.empty(2, 0, 16, 2, 2, 2, dtype=torch.float16, device=DEV))
    x = torch.zeros(3, 0, 128, device=DEV).bfloat16()
    slots = torch.arange(3, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    for f in (lambda: K.kv4_write(x, x, none, slots), lambda: K.kv4_read(none, slots),
              lambda: K.paged_attention_kv4(torch.zeros(1, 4, 128, device=DEV).bfloat16(), none, torch.zeros(1, 1, **i32),
                                            torch.ones(1, **i32))):
        with pytest.raises(RuntimeError, match="KV head"):
            f()
