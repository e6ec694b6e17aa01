"""8-bit KV cache on the GPU: bytes against the definition, attention against 64 bits."""

import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8  # half a step of bf16, relative


def _rows(T, H, hd, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, H, hd, generator=g) * spread * torch.exp(0.5 * torch.randn(H, hd, generator=g))).bfloat16()


def _pair(pages, H, page, hd):
    from meshy_b200.ops.kv8 import kv8_empty

    return kv8_empty(pages, H, page, hd, "cpu"), kv8_empty(pages, H, page, hd, "cuda")


def _same(cpu, gpu):
    for a, b, name in zip(cpu, gpu, cpu._fields):
        b = b.cpu()
        if a.dtype.is_floating_point:
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)), name
        else:
            assert torch.equal(a, b), name


def _write(cpu, gpu, k, v, slots, keep=True):
    from meshy_b200.ops.kv8 import kv8_read, kv8_write

    want = kv8_write(k, v, cpu, slots, keep=True)
    got = kv8_write(k.cuda(), v.cuda(), gpu, slots.cuda(), keep=keep)
    if keep:
        for a, b in zip(want, got):
            assert torch.equal(a.nan_to_num(7.0), b.cpu().nan_to_num(7.0))
    for a, b in zip(kv8_read(cpu, slots, torch.bfloat16), kv8_read(gpu, slots.cuda())):
        assert torch.equal(a.nan_to_num(7.0), b.cpu().nan_to_num(7.0))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T, H, page", [(1, 1, 16), (5, 2, 16), (16, 8, 64), (100, 3, 32), (700, 5, 48), (3001, 2, 128)])
def test_prompt_bytes(T, H, page, hd):
    pages = -(-T // page) + 2
    cpu, gpu = _pair(pages, H, page, hd)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1))
    at = torch.arange(T)
    slots = order[at // page] * page + at % page
    k, v = _rows(T, H, hd), _rows(T, H, hd, 1, 30.0)
    _write(cpu, gpu, k, v, slots)
    _same(cpu, gpu)
    # the next prompt in the same pages starts the blocks anew
    _write(cpu, gpu, v, k, slots, keep=False)
    _same(cpu, gpu)


@pytest.mark.parametrize("hd", [64, 128])
def test_appended_tokens_requantise(hd):
    H, page, rows = 3, 32, 40
    cpu, gpu = _pair(rows + 1, H, page, hd)
    rng = random.Random(2)
    length = [0] * rows
    for step in range(40):
        who = sorted(rng.sample(range(rows), rng.randint(1, rows)))
        slots = torch.tensor([(r + 1) * page + length[r] % page for r in who])
        spread = 2.0 ** torch.tensor([float(rng.randint(-8, 8)) for _ in who])
        k = (_rows(len(who), H, hd, step).float() * spread[:, None, None]).bfloat16()
        v = (_rows(len(who), H, hd, 100 + step).float() / spread[:, None, None]).bfloat16()
        _write(cpu, gpu, k, v, slots, keep=bool(step % 2))
        _same(cpu, gpu)
        for r in who:
            length[r] += 1
    # the same token again changes nothing
    before = [x.clone() for x in gpu]
    _write(cpu, gpu, k, v, slots)
    assert all(torch.equal(a, b) for a, b in zip(before, gpu))


def test_runs_in_any_order_and_slots_outside():
    H, page, hd = 2, 16, 64
    cpu, gpu = _pair(6, H, page, hd)
    parts = []
    rng = random.Random(4)
    for b in (3, 1, 5, 2):  # blocks in any order, their rows too, some of them left out
        at = rng.sample(range(16), rng.randint(1, 16))
        parts += [b * 16 + p for p in at] + [-1, 6 * 16, 1 << 40]
    slots = torch.tensor([-5] * 40 + parts + [-1] * 3)
    k, v = _rows(len(slots), H, hd), _rows(len(slots), H, hd, 1)
    _write(cpu, gpu, k, v, slots)
    _same(cpu, gpu)
    assert int(gpu.k[0].sum()) == 0 and int(gpu.k[4].sum()) == 0


@pytest.mark.parametrize("H, hd", [(1, 64), (2, 128), (8, 128), (11, 64), (70, 64)])
@pytest.mark.parametrize("T", [250, 600, 1500])
def test_many_rows_in_runs_of_any_length(T, H, hd):
    """A row to a block, whole blocks and anything between, in one call: twice, so that the second appends to blocks."""
    rng = random.Random(T + H)
    page, pages = 32, T // 2 + 2
    cpu, gpu = _pair(pages, H, page, hd)
    blocks = [b for b in range(2, 2 * pages)]
    rng.shuffle(blocks)
    most = rng.choice([1, 3, 16])
    runs, slots = [], []
    while len(slots) < T:
        first, n = rng.choice([0, 0, 5]), min(rng.randint(1, most), 8, T - len(slots))
        runs.append((blocks.pop(), first + n))
        slots += [runs[-1][0] * 16 + p for p in range(first, first + n)]
    _write(cpu, gpu, _rows(T, H, hd), _rows(T, H, hd, 1), torch.tensor(slots))
    _same(cpu, gpu)
    slots = [b * 16 + p for b, p in runs]  # the next token of each
    n = len(slots)
    spread = 2.0 ** torch.tensor([float(rng.randint(-2, 2)) for _ in slots])[:, None, None]
    k, v = ((_rows(n, H, hd, 2 + i).float() * spread).bfloat16() for i in range(2))
    _write(cpu, gpu, k, v, torch.tensor(slots), keep=False)
    _same(cpu, gpu)


def test_values_far_and_not_finite():
    H, page, hd = 2, 16, 128
    cpu, gpu = _pair(12, H, page, hd)
    k = torch.zeros(16 * 11, H, hd).bfloat16()
    v = _rows(16 * 11, H, hd)
    blocks = k.view(11, 16, H, hd)
    blocks[1] = 2.0 ** -130                                    # below the smallest scale
    blocks[2, 3, 0, 5] = 2.0 ** -100
    blocks[3] = _rows(16, H, hd, 3, 1e30)
    blocks[4, 0, 0, 0], blocks[4, 2, 0, 1] = math.inf, -math.inf
    blocks[5, 7, 1, 9] = math.nan
    blocks[6] = torch.finfo(torch.bfloat16).max
    blocks[7, :, :, ::2], blocks[7, :, :, 1::2] = 1.0, 0.5     # halves of the step
    blocks[8] = _rows(16, H, hd, 5) * 2.0 ** -126
    blocks[9, 0] = -3.0
    slots = torch.arange(16 * 11) + 16
    _write(cpu, gpu, k, v, slots)
    _same(cpu, gpu)
    # a NaN that is appended, and one that a new first token clears
    _write(cpu, gpu, blocks[5, 7:8].clone(), v[:1], torch.tensor([4 * 16 + 3]))
    _same(cpu, gpu)
    _write(cpu, gpu, v[:1], v[1:2], torch.tensor([6 * 16]))
    _same(cpu, gpu)


def test_scales_of_every_magnitude():
    """All 128 mantissas of a bf16 maximum over the exponents: scales equal to the last bit, in fresh and in kept blocks."""
    tops = torch.arange(0x0080, 0x7F80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    n = len(tops)
    cpu, gpu = _pair(n, 1, 16, 64)
    x = torch.zeros(n, 1, 64).bfloat16()
    x[:, 0, 5], x[:, 0, 6], x[:, 0, 7] = tops, -tops / 2, tops / 3
    slots = torch.arange(n) * 16
    from meshy_b200.ops import reference as ref

    # (the definition over all blocks at once; the block-by-block one takes minutes here)
    r = ref.kv8_steps(tops.float())
    from meshy_b200.ops.kv8 import kv8_write

    kv8_write(x.cuda(), x.cuda(), gpu, slots.cuda())
    assert torch.equal(gpu.scale[:, 0, 0, 0].cpu(), 1.0 / r)
    level = (x[:, 0].float().clamp(-2.0 ** 126, 2.0 ** 126) * r[:, None]).round() + 128
    assert torch.equal(gpu.k[:, 0, 0].cpu(), level.to(torch.uint8))
    # a smaller token keeps r, which is found again from the scale
    kv8_write(x.cuda() * 0, x.cuda() * 0, gpu, slots.cuda() + 1)
    assert torch.equal(gpu.scale[:, 0, 0, 1].cpu(), 1.0 / r) and torch.equal(gpu.k[:, 0, 0].cpu(), level.to(torch.uint8))


def test_repeated_slots_stay_inside():
    """Idle rows all name one slot: it holds one of them, nothing else is touched."""
    from meshy_b200.ops.kv8 import kv8_empty, kv8_read, kv8_write

    c = kv8_empty(4, 2, 16, 64, "cuda")
    k, v = _rows(200, 2, 64).cuda(), _rows(200, 2, 64, 1).cuda()
    slots = torch.zeros(200, dtype=torch.int64, device="cuda")
    slots[:3] = torch.tensor([20, 21, 22])
    kv8_write(k, v, c, slots)
    want = kv8_empty(4, 2, 16, 64, "cuda")
    kv8_write(k[:3], v[:3], want, slots[:3])
    for a, b in zip(c, want):
        assert torch.equal(a[1:], b[1:])
    assert int(c.k[0, :, 1:].sum()) == 0
    assert bool(kv8_read(c, slots[3:4])[0].isfinite().all())


def test_strided_rows_and_none():
    from meshy_b200.ops.kv8 import kv8_empty, kv8_read, kv8_write

    wide = torch.randn(24, 7, 130, device="cuda").bfloat16()
    slots = torch.arange(24, device="cuda")
    for k in (wide[:, 2:4, :64], wide[:, 2:4, 1:65], wide.transpose(0, 1)[:2, :, :64].transpose(0, 1),
              wide.float().transpose(1, 2)[:, :64, 3:5].transpose(1, 2).bfloat16()):
        a, b = kv8_empty(2, 2, 16, 64, "cuda"), kv8_empty(2, 2, 16, 64, "cuda")
        kv8_write(k, k, a, slots)
        kv8_write(k.contiguous(), k.contiguous(), b, slots)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert kv8_write(k[:0], k[:0], a, slots[:0]) is None
    assert kv8_write(k[:0], k[:0], a, slots[:0], keep=True)[0].shape == (0, 2, 64)
    assert kv8_read(a, slots[:0])[0].shape == (0, 2, 64)


# ── attention ────────────────────────────────────────────────────────────────

def _filled(lens, Hkv, hd, page, seed=0, spread=1.0, extra=3):
    """A cache with the rows' tokens on shuffled pages, NaN scales and any bytes elsewhere; (cache, block table)."""
    from meshy_b200.ops.kv8 import kv8_empty, kv8_write

    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra
    c = kv8_empty(pages, Hkv, page, hd, "cuda")
    g = torch.Generator().manual_seed(seed)
    for x in (c.k, c.v):
        x.copy_(torch.randint(0, 256, x.shape, generator=g, dtype=torch.uint8))
    c.scale.fill_(math.nan)
    order = torch.randperm(pages, generator=g).tolist()
    bt = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for i, (n, p) in enumerate(zip(lens, need)):
        bt[i, :p] = torch.tensor(order[at:at + p], dtype=torch.int32)
        at += p
        if n:
            t = torch.arange(n)
            slots = bt[i, t // page].long() * page + t % page
            kv8_write(_rows(n, Hkv, hd, seed + 2 * i + 1, spread).cuda(), _rows(n, Hkv, hd, seed + 2 * i + 2).cuda(), c,
                      slots.cuda())
    return c, bt.cuda()


def _exact(q, c, bt, lens, scale):
    """The attention in 64 bits, the sum of p |v|, how large the scores' terms are, and the sum of p a (a step of V)."""
    B, Hq, hd = q.shape
    Hkv, page = c.k.shape[1], c.k.shape[2]
    out = torch.zeros(B, Hq, hd, dtype=torch.float64, device="cuda")
    size, terms = torch.zeros_like(out), torch.zeros(B, Hq, 1, dtype=torch.float64, device="cuda")
    step = torch.zeros_like(terms)
    for b, n in enumerate(lens):
        t = torch.arange(max(0, min(n, bt.shape[1] * page)), device="cuda")
        pg = bt[b, t // page].long()
        there = (pg >= 0) & (pg < c.k.shape[0])
        pg, off = pg[there], (t % page)[there]
        if not pg.numel():
            continue
        for h in range(Hq):
            hk = h // (Hq // Hkv)
            a = c.scale[pg, hk, off // 16].double()
            k = (c.k[pg, hk, off].double() - 128) * a[:, :1]
            v = (c.v[pg, hk, off].double() - 128) * a[:, 1:]
            p = torch.softmax(k @ q[b, h].double() * scale, 0)
            out[b, h], size[b, h] = p @ v, p @ v.abs()
            terms[b, h] = 255 * a[:, 0].max() * q[b, h].double().abs().sum() * abs(scale)
            step[b, h] = p @ a[:, 1]
    return out, size, terms, step


def _check(q, c, bt, lens, scale=None):
    from meshy_b200.ops.kv8 import paged_attention_kv8

    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = paged_attention_kv8(q, c, bt, sl, scale)
    want, size, terms, step = _exact(q, c, bt, lens, scale if scale is not None else 1 / math.sqrt(q.shape[-1]))
    # bf16 output; a weight times its value's scale has fp16's 11 bits (half a step 2^-11, relative); scores are fp32
    # sums of 10 steps over terms of at most ``terms``, which moves a weight by twice that; exponentials 2^-20
    n = max(lens)
    weights = 2.0 ** -11 + 2 * (10 * 2.0 ** -23 * terms + 2.0 ** -20)
    # The output's fp32 sums: a block's two products add 2 x 17 numbers, each cut at 2^-24 of the largest, which is at
    # most the sum so far (a warp sums n / 128 blocks) or the bytes' offset, 128 x (x = p a), of the up to 16 blocks for
    # which it is taken out together. And an x far below the largest one, 2^11, is off by up to 2^-25, that is 2^-36 of
    # it, times at most 127.
    weights = weights + 34 * 2.0 ** -24 * (n / 128 + 1)
    low = (34 * 128 * 16 * 2.0 ** -24 + n * 127 * 2.0 ** -36) * step
    off, bound = (got.double() - want).abs(), BF16 * want.abs() + weights * size + low + 1e-30
    assert bool((off <= bound).all()), f"off by {(off / bound).max().item():.3g} of the bound"
    return got


def _q(B, Hq, hd, seed=9):
    return torch.randn(B, Hq, hd, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").bfloat16()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 48, 64, 128])
@pytest.mark.parametrize("Hq, Hkv", [(1, 1), (12, 2), (14, 2), (8, 8), (24, 2)])
def test_attention_over_lengths(hd, page, Hq, Hkv):
    lens = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 300, 511, 1000, 0]
    c, bt = _filled(lens, Hkv, hd, page)
    _check(_q(len(lens), Hq, hd), c, bt, lens)


@pytest.mark.parametrize("hd, page, Hq, Hkv, lens", [
    (128, 64, 12, 2, [700]), (128, 64, 16, 2, [20011]), (64, 16, 14, 2, [5001, 0, 17, 3333]),
    (128, 64, 32, 8, [900, 1500, 1, 1024]), (128, 16, 6, 1, [4096] * 5), (128, 128, 16, 2, [9000, 1] * 3),
    (64, 64, 4, 2, [2048] * 40), (128, 64, 12, 2, list(range(1, 8000, 211))),
    (64, 32, 8, 8, [(37 * i) % 900 for i in range(300)]),
], ids=lambda x: str(x)[:24])
def test_attention_over_shapes(hd, page, Hq, Hkv, lens):
    c, bt = _filled(lens, Hkv, hd, page)
    _check(_q(len(lens), Hq, hd), c, bt, lens)


@pytest.mark.parametrize("hd", [64, 128])
def test_every_token_counts_once(hd):
    """Equal scores: the output is the mean of V, which names each token."""
    from meshy_b200.ops.kv8 import KV8Cache, paged_attention_kv8

    page, Hkv = 16, 2
    lens = [1, 5, 16, 100, 1023, 2500, 7001, 33, 64]
    c, bt = _filled(lens, Hkv, hd, page)
    q = torch.zeros(len(lens), 4, hd, device="cuda").bfloat16()
    got = paged_attention_kv8(q, KV8Cache(*c), bt, torch.tensor(lens, dtype=torch.int32, device="cuda")).double()
    want, size, _, step = _exact(q, c, bt, lens, 1.0)
    # weights are all 1: times a scale, rounded to 11 bits (one rounding for the 16 tokens of a block); sums as above
    sums = 34 * 2.0 ** -24 * (max(lens) / 128 + 1) * size + 34 * 128 * 16 * 2.0 ** -24 * step
    assert bool(((got - want).abs() <= BF16 * want.abs() + 2.0 ** -11 * size + sums).all())


def test_pages_and_lengths_outside():
    hd, page, Hkv = 128, 16, 2
    lens = [100, 70, 33, 16, 20]
    c, bt = _filled(lens, Hkv, hd, page)
    bt[0, 2], bt[1, 0], bt[1, 4], bt[2, :] = -1, 1 << 30, c.k.shape[0], -9
    _check(_q(5, 12, hd), c, bt, lens)
    # lengths past the table end with it (row 4 has pages to its end), those below zero are empty
    bt[3, :], bt[4, :] = bt[3, 0], bt[4, 0]
    lens[3], lens[4] = (1 << 31) - 1, bt.shape[1] * page
    got = _check(_q(5, 12, hd), c, bt[:, :1], [16, 70, 33, (1 << 31) - 1, -5])
    assert float(got[4].abs().sum()) == 0.0 and float(got[2].abs().sum()) == 0.0


def test_scores_far_apart():
    """Weights from one to nothing, values of no weight that are far larger, values of many sizes."""
    from meshy_b200.ops.kv8 import kv8_write

    hd, page, Hkv = 128, 64, 2
    lens = [2000, 555]
    for spread in (1.0, 40.0, 1000.0):
        c, bt = _filled(lens, Hkv, hd, page, seed=5, spread=spread)
        _check(_q(2, 16, hd), c, bt, lens, scale=0.7)
    c, bt = _filled(lens, Hkv, hd, page, seed=5)
    for i, n in enumerate(lens):
        t = torch.arange(n)
        slots = bt[i].cpu()[t // page].long() * page + t % page
        size = 10.0 ** (torch.arange(n) // 16 % 17 - 8).float()[:, None, None]
        for s in (size, size.flip(0), 1e-30 * size.clamp(max=1.0), torch.where(size > 1, 0.0, size)):
            kv8_write(_rows(n, Hkv, hd, 3, 4.0).cuda(), (_rows(n, Hkv, hd, 4).float() * s).bfloat16().cuda(), c, slots.cuda())
            if float(s.max()) > 1e-20:
                _check(_q(2, 16, hd), c, bt, lens, scale=0.7)


def test_strided_queries_and_a_part_of_a_table():
    from meshy_b200.ops.kv8 import paged_attention_kv8

    lens = [40, 100, 7]
    c, bt = _filled(lens, 2, 64, 16)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    wide = torch.randn(3, 20, 100, device="cuda").bfloat16()
    wbt = torch.cat((bt, bt), 1)
    for q in (wide[:, 3:7, :64], wide[:, 3:7, 3:67], wide[:, ::5, 8:72]):
        want = paged_attention_kv8(q.contiguous(), c, bt, sl)
        assert torch.equal(paged_attention_kv8(q, c, bt, sl), want)
        assert torch.equal(paged_attention_kv8(q, c, wbt[:, :bt.shape[1]], sl), want)


def test_captured_graphs_follow_lengths_and_share_nothing():
    """Two graphs captured on one stream, replayed at the same time on others."""
    from meshy_b200.ops.kv8 import paged_attention_kv8

    lens = [9000, 1, 3000, 0]
    c, bt = _filled(lens, 2, 128, 64)
    qs = [_q(4, 12, 128, s) for s in (1, 2)]
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([paged_attention_kv8(q, c, bt, sl) for _ in range(3)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in qs]
    for new in (lens, [17, 8000, 0, 2000], [0, 0, 0, 0], [9000, 1, 3000, 0]):
        now = torch.tensor([min(a, b) for a, b in zip(new, lens)], dtype=torch.int32)
        sl.copy_(now)
        torch.cuda.synchronize()
        for _ in range(20):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for q, o in zip(qs, outs):
            want = _check(q, c, bt, now.tolist())
            assert all(torch.equal(x, want) for x in o)


def test_many_calls_on_streams_at_once():
    from meshy_b200.ops.kv8 import paged_attention_kv8

    lens = [5000, 300, 4000]
    c, bt = _filled(lens, 2, 128, 64)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs = [_q(3, 16, 128, s) for s in range(4)]
    want = [paged_attention_kv8(q, c, bt, sl) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = []
    for _ in range(10):
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(paged_attention_kv8(q, c, bt, sl))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 4]) for i, g in enumerate(got))


def test_calls_from_several_threads():
    """Each on a stream of its own, calls and captured graphs that come and go."""
    import threading

    from meshy_b200.ops.kv8 import paged_attention_kv8

    lens = [900, 30, 2000]
    c, bt = _filled(lens, 2, 64, 32)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qs = [_q(3, 12, 64, s) for s in range(4)]
    want = [paged_attention_kv8(q, c, bt, sl) for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for turn in range(6):
                    got = paged_attention_kv8(qs[i], c, bt, sl)
                    graph = torch.cuda.CUDAGraph()
                    graph.capture_begin(capture_error_mode="thread_local")
                    held = paged_attention_kv8(qs[i], c, bt, sl)
                    graph.capture_end()
                    graph.replay()
                    s.synchronize()
                    if not (torch.equal(got, want[i]) and torch.equal(held, want[i])):
                        wrong.append((i, turn))
                    del graph, held
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not any(t.is_alive() for t in threads) and not wrong, wrong


@pytest.mark.parametrize("qscale", [0.0, 1e-30, 1e-6, 200.0, 1e30])
def test_query_scales(qscale):
    from meshy_b200.ops.kv8 import paged_attention_kv8

    lens = [900, 64]
    c, bt = _filled(lens, 2, 128, 64, seed=6, spread=1.0 / max(qscale, 1.0))
    q = (_q(2, 12, 128).float() * qscale).bfloat16()
    for scale in (None, 0.25 / max(1.0, qscale) * 1.7):
        if qscale < 1e20 or scale:
            _check(q, c, bt, lens, scale)
    if qscale < 1e20:
        _check(q, c, bt, lens, -0.3 / max(1.0, qscale))
    q[1, 3] = 0.0  # a head of zeros beside others: the mean of V
    _check(q, c, bt, lens, 0.25 / max(1.0, qscale))
    # a NaN in one head stays there
    q[0, 2, 7] = math.nan
    out = paged_attention_kv8(q, c, bt, torch.tensor(lens, dtype=torch.int32, device="cuda"), 0.25 / max(1.0, qscale))
    assert bool(out[0, 2].isnan().all()) and int(out.isnan().any(-1).sum()) == 1


@pytest.mark.parametrize("peak", [0, 40000, 65535])
def test_a_long_tail_keeps_its_mass(peak):
    """One key ahead of 65535 others by a factor 2^22: their common weight, 2^-6, has to arrive. (In the peak's block the
    others' values are quantised beside zeros: the same scale.)"""
    from meshy_b200.ops.kv8 import kv8_empty, kv8_write

    L, hd = 65536, 128
    k = torch.zeros(L, 1, hd, device="cuda")
    k[peak, 0, 0] = 16.0
    v = torch.full((L, 1, hd), 10.0, device="cuda")
    v += (torch.arange(hd, device="cuda") % 2) * 2
    v[peak] = 0
    c = kv8_empty(L // 64, 1, 64, hd, "cuda")
    kv8_write(k.bfloat16(), v.bfloat16(), c, torch.arange(L, device="cuda"))
    q = torch.zeros(1, 2, hd, device="cuda").bfloat16()
    q[..., 0] = 1.0
    _check(q, c, torch.arange(L // 64, dtype=torch.int32, device="cuda")[None], [L], 22 * math.log(2) / 16)


@pytest.mark.parametrize("L", [700, 20000])
@pytest.mark.parametrize("every", [0, 256, 32])
def test_small_values_beside_blocks_of_large_ones(L, every):
    """Values that carry the result beside blocks of next to no weight whose values are ten thousand times as large, and
    below peaks that have no values at all."""
    from meshy_b200.ops.kv8 import kv8_empty, kv8_write

    hd = 128
    g = torch.Generator(device="cuda").manual_seed(12)
    t = torch.arange(L, device="cuda")
    k = torch.zeros(L, 1, hd, device="cuda")
    v = 10 + 4 * torch.rand(L, 1, hd, generator=g, device="cuda")
    k[t % 256 == 21, 0, 0] = 16.0                # a factor 2^22 ahead of the others
    v[t % 256 == 21] = 0
    if every:
        far = t // 16 * 16 % every == 0
        k[far, 0, 0] = -64.0                     # 2^-88 of the others
        v[far] = 65504.0 * (torch.arange(hd, device="cuda") % 2 * 2 - 1)
    q = torch.zeros(1, 2, hd, device="cuda").bfloat16()
    q[..., 0] = 1.0
    bt = torch.arange(-(-L // 64), dtype=torch.int32, device="cuda")[None]
    c = kv8_empty(bt.shape[1], 1, 64, hd, "cuda")
    kv8_write(k.bfloat16(), v.bfloat16(), c, t)
    _check(q, c, bt, [L], 22 * math.log(2) / 16)


def test_rising_scores():
    """Every block's maximum above the last: the reference moves at every step, late keys carry the weight."""
    from meshy_b200.ops.kv8 import kv8_empty, kv8_write

    L, hd = 5000, 128
    k = torch.zeros(L, 2, hd, device="cuda")
    k[:, :, 0] = torch.arange(L, device="cuda")[:, None] * (60.0 / L)
    v = torch.randn(L, 2, hd, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    c = kv8_empty(-(-L // 16), 2, 16, hd, "cuda")
    kv8_write(k.bfloat16(), v.bfloat16(), c, torch.arange(L, device="cuda"))
    bt = torch.arange(-(-L // 16), dtype=torch.int32, device="cuda")[None]
    for sign in (1.0, -1.0):
        q = torch.zeros(1, 4, hd, device="cuda").bfloat16()
        q[..., 0] = sign * 8
        _check(q, c, bt, [L])


def test_nan_key_reaches_its_row_only():
    from meshy_b200.ops.kv8 import kv8_write, paged_attention_kv8

    lens = [300, 300]
    c, bt = _filled(lens, 2, 128, 64)
    slot = int(bt[0, 2]) * 64 + 7
    bad = torch.full((1, 2, 128), math.nan, device="cuda").bfloat16()
    kv8_write(bad, torch.zeros_like(bad), c, torch.tensor([slot], device="cuda"))
    q = _q(2, 12, 128)
    out = paged_attention_kv8(q, c, bt, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert bool(out[0].isnan().all())
    assert torch.equal(out[1:], _check(q[1:], c, bt[1:], lens[1:]))


def test_length_at_the_end_of_32_bits():
    """A table that spans 2^31 tokens and a length of 2^31 - 1: rounding it up to whole units must not wrap."""
    from meshy_b200.ops.kv8 import paged_attention_kv8

    c, bt = _filled([200], 1, 128, 64)
    wide = torch.full((1, (1 << 25) + 1), -1, dtype=torch.int32, device="cuda")
    wide[:, :2] = bt[:, :2]
    q = _q(1, 2, 128)
    out = paged_attention_kv8(q, c, wide, torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    want, size, terms, step = _exact(q, c, bt, [128], 1 / math.sqrt(128))
    bound = BF16 * want.abs() + (2.0 ** -11 + 2 * (10 * 2.0 ** -23 * terms + 2.0 ** -20)) * size + 34 * 128 * 16 * 2.0 ** -24 * step
    assert bool(((out.double() - want).abs() <= bound).all())


def test_offsets_beyond_32_bits():
    from meshy_b200.ops.kv8 import KV8Cache, kv8_read, kv8_write

    page, H, hd = 64, 2, 128
    P = (1 << 32) // (H * page * hd) + 64  # more than 2^32 bytes of K
    c = KV8Cache(torch.empty(P, H, page, hd, dtype=torch.uint8, device="cuda"),
                 torch.empty(P, H, page, hd, dtype=torch.uint8, device="cuda"),
                 torch.empty(P, H, page // 16, 2, device="cuda"))
    pages = torch.tensor([P - 1, 0, P - 40], device="cuda")
    t = torch.arange(150, device="cuda")
    slots = pages[t // page] * page + t % page
    x = _rows(150, H, hd, 9).cuda()
    ko, vo = kv8_write(x, -x, c, slots, keep=True)
    k, v = kv8_read(c, slots)
    assert torch.equal(k, ko) and torch.equal(v, vo) and torch.equal(k, -v) and float((k - x).abs().max()) < 0.1
    _check(_q(1, 12, hd), c, pages.int()[None], [150])


def test_rows_beyond_32_bits():
    """More than 2^31 channels in one call: its last rows hold what a call on them alone gives."""
    from meshy_b200.ops.kv8 import kv8_empty, kv8_read, kv8_write

    H, hd, page, T = 16, 128, 64, (1 << 20) + 640
    base = _rows(997, H, hd, 3).cuda()
    x = base[torch.arange(T, device="cuda") % 997]
    c = kv8_empty(T // page, H, page, hd, "cuda")
    slots = torch.arange(T, device="cuda")
    ko, vo = kv8_write(x, x, c, slots, keep=True)
    k, v = kv8_read(c, slots)
    tail = kv8_empty(16, H, page, hd, "cuda")
    want, _ = kv8_write(x[-1024:], x[-1024:], tail, torch.arange(1024, device="cuda"), keep=True)
    for got in (ko, vo, k, v):
        assert torch.equal(got[-1024:], want)
    assert torch.equal(ko, k) and torch.equal(vo, v) and torch.equal(c.k[-16:], tail.k) and torch.equal(c.scale[-16:], tail.scale)


def test_workspace_grows_with_the_segments():
    """More segments than the first counters hold (16384), on a stream that has used the smaller ones, and in a capture."""
    from meshy_b200.ops.kv8 import paged_attention_kv8

    lens = torch.randint(0, 40, (2100,), generator=torch.Generator().manual_seed(4)).tolist()
    small_lens = [40, 3000]
    c, bt = _filled(lens[:64], 8, 64, 16)
    bt = bt.repeat(33, 1)[:2100]
    sl = torch.tensor((lens[:64] * 33)[:2100], dtype=torch.int32, device="cuda")
    sc, sbt = _filled(small_lens, 8, 64, 16)
    ssl = torch.tensor(small_lens, dtype=torch.int32, device="cuda")
    q, sq = _q(2100, 8, 64), _q(2, 8, 64)

    def step():
        return [paged_attention_kv8(sq, sc, sbt, ssl), paged_attention_kv8(q, c, bt, sl), paged_attention_kv8(q, c, bt, sl),
                paged_attention_kv8(sq, sc, sbt, ssl)]

    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        a = step()
    s.synchronize()
    assert torch.equal(a[0], a[3]) and torch.equal(a[1], a[2])
    _check(sq, sc, sbt, small_lens)
    want, size, terms, step_ = _exact(q[:64], c, bt[:64], lens[:64], 1 / 8)
    bound = BF16 * want.abs() + (2.0 ** -11 + 2 * (10 * 2.0 ** -23 * terms + 2.0 ** -20)) * size + 34 * 128 * 16 * 2.0 ** -24 * step_
    assert bool(((a[1][:64].double() - want).abs() <= bound).all())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b = step()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_graphs_come_and_go():
    """Graphs that are made, replayed and dropped hand their workspaces on; a capture that fails hands its back too."""
    from meshy_b200.ops.kv8 import paged_attention_kv8

    lens = [3000, 5, 700]
    c, bt = _filled(lens, 2, 128, 64)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = _q(3, 12, 128)
    want = paged_attention_kv8(q, c, bt, sl)
    free = []
    for i in range(12):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = paged_attention_kv8(q, c, bt, sl)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del g, out
        if i == 3:
            with pytest.raises(RuntimeError):
                with torch.cuda.graph(torch.cuda.CUDAGraph()):
                    paged_attention_kv8(q, c, bt, sl)
                    paged_attention_kv8(q[:, :5], c, bt, sl)
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        free.append(torch.cuda.mem_get_info()[0])
    assert min(free[6:]) >= free[5] - (4 << 20)  # 1.3 MB each: those of the dropped graphs were taken again
    assert torch.equal(paged_attention_kv8(q, c, bt, sl), want)


def test_a_step_together():
    """Rotary, maps, write and attention as a decode step chains them, against the functions of the CPU."""
    from meshy_b200.ops import kv8, paging, rotary

    Hq, Hkv, hd, page, B = 4, 2, 64, 16, 3
    rope = rotary.Rope(hd, 1e4, 32, True, {"rope_type": "linear", "factor": 2.0})
    lens = [20, 1, 47]
    T = sum(lens)
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * hd, generator=g).bfloat16()
    step = torch.randn(4, B, (Hq + 2 * Hkv) * hd, generator=g).bfloat16()

    def run(dev):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        c = kv8.kv8_empty(16, Hkv, page, hd, dev)
        bt, rows = torch.zeros(5, 4, dtype=torch.int32, device=dev), i32([4, 0, 2])
        paging.assign_pages(bt, rows, i32([0] * B), i32([-(-(n + 4) // page) for n in lens]), i32(range(1, 12)))
        m = paging.token_maps(bt, rows, i32([0] * B), i32(lens), T, page)
        _, k, v = rotary.qkv_rotary(qkv.to(dev), m.positions, rope, Hq, Hkv)
        outs = [*kv8.kv8_write(k, v, c, m.slots, keep=True)]
        for s in range(4):
            now = i32([n + s for n in lens])
            m = paging.token_maps(bt, rows, now, i32([1] * B), B, page)
            q, k, v = rotary.qkv_rotary(step[s].to(dev), m.positions, rope, Hq, Hkv)
            kv8.kv8_write(k, v, c, m.slots)
            outs.append(kv8.paged_attention_kv8(q, c, bt[rows.long()], now + 1))
        return [x.cpu().double() for x in outs]

    for a, b in zip(run("cpu"), run("cuda")):
        # bf16 at every stage: a channel that falls on the other side of a rounding moves a value by a step of the cache
        assert float((a - b).abs().max()) <= 0.06 and float((a - b).abs().mean()) <= 2.0 ** -8


def test_refusals():
    from meshy_b200.ops.kv8 import KV8Cache, kv8_empty, kv8_read, kv8_write, paged_attention_kv8

    c = kv8_empty(4, 2, 16, 64, "cuda")
    k = torch.zeros(3, 2, 64, device="cuda").bfloat16()
    s = torch.arange(3, device="cuda")
    bt, sl = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    for a in ((k.float(), k, c, s), (k, k[:, :1], c, s), (k[:2], k[:2], c, s), (k, k, c, s.int()), (k, k, c, s.cpu()),
              (k[..., :32], k[..., :32], c, s), (k, k, KV8Cache(c.k, c.v[:2], c.scale), s),
              (k, k, KV8Cache(c.k, c.v, c.scale[:2]), s), (k, k, KV8Cache(c.k, c.v, c.scale.half()), s),
              (k, k, KV8Cache(c.k[:, :, :8], c.v[:, :, :8], c.scale), s),
              (k, k, KV8Cache(c.k.transpose(2, 3).contiguous().transpose(2, 3), c.v, c.scale), s)):
        with pytest.raises(RuntimeError):
            kv8_write(*a)
    with pytest.raises(RuntimeError):
        kv8_read(c, s.int())
    with pytest.raises(ValueError):
        kv8_read(c, s, torch.float32)
    q = torch.zeros(3, 4, 64, device="cuda").bfloat16()
    for a in ((q[:, :3], c, bt, sl), (q.half(), c, bt, sl), (q, c, bt.long(), sl), (q, c, bt, sl.long()), (q, c, bt[:2], sl),
              (q, c, bt, sl[:2]), (q, c, bt.t().contiguous().t(), sl), (q, c, bt.cpu(), sl)):
        with pytest.raises(RuntimeError):
            paged_attention_kv8(*a)
    for hd, page, n in ((32, 16, 2), (64, 8, 2), (64, 16, 0), (64, 0, 2)):
        with pytest.raises(ValueError):
            kv8_empty(2, n, page, hd, "cuda")
