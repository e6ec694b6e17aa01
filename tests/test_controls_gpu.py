"""Logit-control kernels against a plain implementation in 64 bits.

The token state is compared exactly. A controlled logit is at most five fp32 operations on terms that are exact in
fp32, so its error is below 5 * 2^-24 of the sum of the terms' sizes.
"""

import math

import pytest
import torch

from meshy_b200.ops import controls as C

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def _bits_of(words, V):
    sh = torch.arange(32, dtype=torch.int32, device=words.device)
    return ((words.unsqueeze(-1) >> sh) & 1).bool().flatten(-2)[..., :V]


def _state(slots, V, K, seed, masked=True):
    g = _gen(seed)
    ctl = C.LogitControls.create(slots, V, device=DEV, max_bias=K)
    n = min(400, V)
    hist = (torch.rand(slots, n, generator=g, device=DEV) ** 2 * V).long().clamp(max=V - 1)
    cu = torch.arange(slots + 1, dtype=torch.int32, device=DEV) * n
    C.load_tokens(ctl, torch.arange(slots, device=DEV), hist.flatten(), cu, torch.full((slots,), n // 3, dtype=torch.int32, device=DEV))
    pick = lambda vals: torch.tensor(vals, device=DEV)[torch.randint(len(vals), (slots,), generator=g, device=DEV)]
    ctl.repetition.copy_(pick([1.0, 1.3, 0.8]))
    ctl.frequency.copy_(pick([0.0, 0.3, -0.2]))
    ctl.presence.copy_(pick([0.0, 0.7]))
    if K:
        ids = torch.stack([torch.randperm(V, generator=g, device=DEV)[:K] if V >= K else
                           torch.cat([torch.randperm(V, generator=g, device=DEV), torch.full((K - V,), -1, device=DEV)])
                           for _ in range(slots)])
        ids[:, ::3] = -1
        ctl.bias_ids.copy_(ids)
        ctl.bias_vals.copy_(torch.randn(slots, K, generator=g, device=DEV) * 5)
    if masked:
        ctl.mask.copy_(torch.randint(-2 ** 31, 2 ** 31, ctl.mask.shape, generator=g, device=DEV))
        ctl.mask_on.copy_(torch.arange(slots, device=DEV) % 2)
    return ctl


def _expect(z, ctl, slots):
    """fp64 result and the sum of the terms' sizes."""
    out, size = z.double().clone(), z.double().abs()
    V = z.shape[1]
    for b, s in enumerate(slots.tolist()):
        if s < 0:
            continue
        r, f, p = float(ctl.repetition[s]), float(ctl.frequency[s]), float(ctl.presence[s])
        c = ctl.counts[s].double()
        x = out[b]
        x = torch.where(_bits_of(ctl.seen[s], V), torch.where(x > 0, x / r, x * r), x)
        size[b] = torch.maximum(size[b], x.abs()) + abs(f) * c + abs(p) * (c > 0)
        x = x - f * c - p * (c > 0)
        ids = ctl.bias_ids[s].long()
        use = ids >= 0
        x = x.index_add(0, ids[use], ctl.bias_vals[s][use].double())
        size[b].index_add_(0, ids[use], ctl.bias_vals[s][use].double().abs())
        if int(ctl.mask_on[s]):
            x = x.masked_fill(~_bits_of(ctl.mask[s], V), -math.inf)
        out[b] = x
    return out, size


def _check(out, want, size):
    assert out.dtype == torch.float32
    fin = want.isfinite()
    assert torch.equal(out[~fin].isnan(), want[~fin].isnan())
    assert torch.equal(out[~fin].nan_to_num(), want[~fin].float().nan_to_num())
    err = (out.double() - want).abs()[fin]
    assert bool((err <= 5 * 2 ** -24 * size[fin]).all()), f"largest error {float(err.max())}"


@pytest.mark.parametrize("V", [1, 31, 32, 33, 100, 2048, 4095, 4097, 32001, 151936])
@pytest.mark.parametrize("B,K,dtype", [(1, 0, torch.float32), (5, 7, torch.float32), (5, 300, torch.bfloat16),
                                       (70, 2, torch.float32)])
def test_controls(V, B, K, dtype):
    slots = B + 3
    ctl = _state(slots, V, K, seed=V + B)
    g = _gen(7)
    z = (torch.randn(B, V, generator=g, device=DEV) * 4).to(dtype)
    ids = torch.randperm(slots, generator=g, device=DEV)[:B]
    if B > 2:
        ids[1] = -1
    want, size = _expect(z, ctl, ids)
    out = torch.full((B, V), 77.0, device=DEV)
    raw = z.clone()
    assert C.apply_logit_controls(z, ctl, ids, out=out) is out and torch.equal(z, raw)
    _check(out, want, size)
    got = C.apply_logit_controls(z, ctl, ids.int())  # fp32: in place
    assert (got.data_ptr() == z.data_ptr()) == (dtype == torch.float32) and torch.equal(got, out)


def test_strided_rows_and_odd_starts():
    V, B = 1001, 4
    ctl = _state(B, V, 5, seed=1)
    ids = torch.arange(B, device=DEV)
    big = torch.randn(B, V + 30, generator=_gen(2), device=DEV)
    for off in (0, 1, 2, 4):
        z = big.clone()[:, off:off + V]
        want, size = _expect(z, ctl, ids)
        dst = torch.full((B, V + 11), 9.0, device=DEV)
        C.apply_logit_controls(z, ctl, ids, out=dst[:, 3:3 + V])
        _check(dst[:, 3:3 + V], want, size)
        assert bool((dst[:, :3] == 9).all()) and bool((dst[:, 3 + V:] == 9).all())
        C.apply_logit_controls(z, ctl, ids)
        _check(z, want, size)


def test_infinite_and_nan_logits():
    V = 64
    ctl = _state(2, V, 0, seed=3, masked=False)
    ctl.mask_on.copy_(torch.tensor([1, 0]))
    ctl.mask.zero_()
    ctl.mask[0, 0] = 0b111
    z = torch.randn(2, V, generator=_gen(4), device=DEV)
    z[:, 1], z[:, 2], z[:, 40], z[:, 41], z[:, 42] = -math.inf, math.nan, math.nan, math.inf, -3.4e38
    want, size = _expect(z, ctl, torch.arange(2, device=DEV))
    out = C.apply_logit_controls(z.clone(), ctl, torch.arange(2, device=DEV))
    assert bool((out[0, 3:] == -math.inf).all()) and bool(out[0, 2].isnan())
    _check(out, want.float().double(), size)


@pytest.mark.parametrize("V", [1, 15, 17, 33, 100, 1009, 4097])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_bits_behind_the_vocabulary_are_no_tokens(V, dtype):
    """Every bit of the seen rows set, those of the last word past V too: nothing outside a row is touched."""
    B = 3
    ctl = _state(B, V, 2 if V > 1 else 0, seed=V)
    ctl.seen.fill_(-1)
    ctl.repetition.fill_(1.3)
    ids = torch.tensor([2, 0, 1], device=DEV)
    z = (torch.randn(B, V, generator=_gen(V), device=DEV) * 4).to(dtype)
    want, size = _expect(z, ctl, ids)
    counts = ctl.counts.clone()
    for pad in (0, 64):  # rows right behind one another, and apart
        room = torch.full((64 + B * (V + pad) + 64,), 7.0, device=DEV)
        out = room[64:64 + B * (V + pad)].view(B, V + pad)[:, :V]
        if dtype == torch.float32:
            out.copy_(z)
            C.apply_logit_controls(out, ctl, ids)
            _check(out, want, size)
            out.fill_(7.0)
        C.apply_logit_controls(z, ctl, ids, out=out)
        _check(out, want, size)
        out.fill_(7.0)
        assert bool((room == 7).all()) and torch.equal(ctl.counts, counts)


def test_mask_that_leaves_nothing():
    ctl = C.LogitControls.create(1, 100, device=DEV, max_bias=0)
    ctl.set_mask(0, torch.zeros(4, dtype=torch.int32))
    out = C.apply_logit_controls(torch.randn(1, 100, device=DEV), ctl, torch.tensor([0], device=DEV))
    assert bool((out == -math.inf).all())


@pytest.mark.parametrize("V", [33, 5000])
def test_counts_the_new_tokens_first(V):
    B = 6
    ctl = _state(8, V, 0, seed=5, masked=False)
    ctl.frequency.fill_(0.5)
    before, seen = ctl.counts.clone(), _bits_of(ctl.seen, V).clone()
    ids = torch.tensor([7, 2, 0, 5, 1, 3], device=DEV)
    tok = torch.tensor([V - 1, 0, -1, 31, V, 32], device=DEV)
    done = torch.tensor([0, 0, 0, 1, 0, 0], dtype=torch.int32, device=DEV)
    z = torch.randn(B, V, generator=_gen(6), device=DEV)
    out = C.apply_logit_controls(z.clone(), ctl, ids, new_tokens=tok, done=done)
    for s, t in ((7, V - 1), (2, 0), (3, 32)):
        before[s, t] += 1
        seen[s, t] = True
    assert torch.equal(ctl.counts, before) and torch.equal(_bits_of(ctl.seen, V), seen)
    _check(out, *_expect(z, ctl, ids))  # with the new counts


@pytest.mark.parametrize("V,lens", [(1, [3]), (33, [0, 1, 200]), (4097, [5000, 17]), (151936, [1, 30000, 0, 2000]), (100003, [64] * 40)])
def test_token_state(V, lens):
    n = len(lens)
    g = _gen(V)
    R = n + 2
    ctl = C.LogitControls.create(R, V, device=DEV, max_bias=0)
    ctl.seen.fill_(-1)
    ctl.counts.fill_(12345)
    slots = torch.randperm(R, generator=g, device=DEV)[:n]
    if n > 2:
        slots[1] = -1
    toks = ((torch.rand(sum(lens), generator=g, device=DEV) ** 3 * (V + 2)).long() - 1)  # -1 and V + 0 occur: ignored
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    npr = torch.tensor([l // 3 for l in lens], dtype=torch.int32, device=DEV)
    C.load_tokens(ctl, slots, toks, cu, npr)
    touched = set()
    for i, s in enumerate(slots.tolist()):
        if s < 0:
            continue
        touched.add(s)
        t = toks[int(cu[i]):int(cu[i + 1])]
        ok = (t >= 0) & (t < V)
        pos = torch.arange(t.numel(), device=DEV) >= int(npr[i])
        assert torch.equal(_bits_of(ctl.seen[s], V), torch.bincount(t[ok], minlength=V)[:V] > 0)
        assert torch.equal(ctl.counts[s].long(), torch.bincount(t[ok & pos], minlength=V))
        pad = _bits_of(ctl.seen[s], 32 * ctl.seen.shape[1])[V:]
        assert not bool(pad.any())
    for s in set(range(R)) - touched:
        assert bool((ctl.counts[s] == 12345).all()) and bool((ctl.seen[s] == -1).all())


def test_graph_replay_counts():
    V = 3000
    ctl = C.LogitControls.create(2, V, device=DEV, max_bias=0)
    ctl.set_slot(0, presence_penalty=1.0)
    z, ids = torch.zeros(2, V, device=DEV), torch.arange(2, device=DEV)
    tok = torch.tensor([5, 6], device=DEV)
    out = torch.empty_like(z)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        C.apply_logit_controls(z, ctl, ids, out=out)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        C.apply_logit_controls(z, ctl, ids, new_tokens=tok, out=out)
    for i in range(3):
        tok[0] = 100 + i
        g.replay()
    torch.cuda.synchronize()
    assert ctl.counts[0].nonzero().flatten().tolist() == [100, 101, 102] and int(ctl.counts[1, 6]) == 3
    assert out[0, 100:103].tolist() == [-1.0] * 3 and float(out[0].sum()) == -3.0


def test_out_apart_from_the_logits_or_the_logits():
    """An output that shares memory with the logits other than entry by entry is refused; rows that take turns are not."""
    V, B = 64, 3
    ctl = _state(B, V, 2, seed=1)
    ids = torch.arange(B, device=DEV)
    room = torch.randn(2 * (B + 1) * V, generator=_gen(2), device=DEV)
    whole = room.clone()
    rows = lambda at, stride, n=B: room.as_strided((n, V), (stride, 1), at)
    for z, out in ((rows(0, V), rows(4, V)), (rows(4, V), rows(0, V)), (rows(0, V), rows(V, V)), (rows(0, V), rows(0, 2 * V)),
                   (rows(0, 2 * V), rows(V - 1, 2 * V)), (rows(0, 2 * V), rows(V + 1, 2 * V)), (rows(V + 4, 2 * V), rows(0, 2 * V + 4)),
                   (room.view(torch.bfloat16)[:B * V].view(B, V), rows(0, V)), (rows(0, V, 1), rows(V - 1, V, 1))):
        with pytest.raises(RuntimeError, match="apart"):
            C.apply_logit_controls(z, ctl, ids[:len(z)], out=out)
    assert torch.equal(room, whole)
    for z, out in ((rows(0, 2 * V), rows(V, 2 * V)), (rows(V, 2 * V), rows(0, 2 * V)), (rows(0, V), rows(B * V, V)),
                   (rows(0, V, 1), rows(V, V, 1))):
        want, size = _expect(z, ctl, ids[:len(z)])
        C.apply_logit_controls(z, ctl, ids[:len(z)], out=out)
        _check(out, want, size)
        room.copy_(whole)


def test_refusals():
    V = 50
    ctl = C.LogitControls.create(2, V, device=DEV, max_bias=0)
    z, ids = torch.zeros(2, V, device=DEV), torch.arange(2, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    tok = torch.zeros(4, dtype=torch.int64, device=DEV)
    cu, npr = torch.tensor([0, 2, 4], **i32), torch.zeros(2, **i32)
    bad = [lambda: C.apply_logit_controls(z.half(), ctl, ids), lambda: C.apply_logit_controls(z[:, :-1], ctl, ids),
           lambda: C.apply_logit_controls(z, ctl, ids.cpu()), lambda: C.apply_logit_controls(z, ctl, ids[:1]),
           lambda: C.apply_logit_controls(z, ctl, ids.float()), lambda: C.apply_logit_controls(z, ctl, ids, new_tokens=ids.int()),
           lambda: C.apply_logit_controls(z, ctl, ids, new_tokens=tok), lambda: C.apply_logit_controls(z, ctl, ids, out=z.double()),
           lambda: C.apply_logit_controls(z.t().contiguous().t(), ctl, ids),
           lambda: C.apply_logit_controls(z.bfloat16(), ctl, ids, out=torch.zeros(1, V, device=DEV).expand(2, V)),
           lambda: C.load_tokens(ctl, ids, tok.int(), cu, npr), lambda: C.load_tokens(ctl, ids, tok, cu.long(), npr),
           lambda: C.load_tokens(ctl, ids, tok, cu[:2], npr), lambda: C.load_tokens(ctl, ids, tok, cu, npr[:1]),
           lambda: C.load_tokens(ctl, ids, tok.cpu(), cu, npr)]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, ValueError)):
            f()
            pytest.fail(f"call {i} was accepted")
    assert C.apply_logit_controls(z[:0], ctl, ids[:0]).shape == (0, V)
    C.load_tokens(ctl, ids[:0], tok[:0], cu[:1], npr[:0])
