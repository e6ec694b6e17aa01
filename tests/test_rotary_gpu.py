"""Rotary kernels (layouts, part of a head, scaled contexts, QK-norm, gradients) against 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8  # half a step of bf16, relative
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
LINEAR = {"rope_type": "linear", "factor": 2.5}


def _rope(hd, rot=None, inter=False, scaling=None, theta=1e4):
    from meshy_b200.ops.rotary import Rope

    return Rope(hd, theta, rot, inter, scaling)


def _inputs(T, Hq, Hkv, hd, norm, seed=0, longest=5000):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * hd, generator=g, device="cuda").bfloat16()
    pos = torch.randint(longest, (T,), generator=g, device="cuda", dtype=torch.int32)
    ws = [(1 + 0.2 * torch.randn(hd, generator=g, device="cuda")).bfloat16() if norm else None for _ in "qk"]
    return qkv, pos, *ws


def _size(x, rope):
    """|a| + |b| of the pair each channel is in (|x| behind the rotated part), times the factor."""
    from meshy_b200.ops import reference as ref

    one = torch.ones(x.shape[0], rope.rotary_dim // 2, dtype=x.dtype, device=x.device) * rope.factor
    a = ref.apply_rotary(x.abs(), one, one, rope)     # |a| - |b| and |b| + |a|
    b = ref.apply_rotary(x.abs(), one, -one, rope)    # |a| + |b| and |b| - |a|
    return torch.maximum(a, b)


def _near(got, want, extra):
    off = (got.double() - want).abs()
    bound = BF16 * want.abs() + extra
    assert bool((off <= bound).all()), f"off by up to {(off / bound.clamp(min=1e-30)).max().item():.3g} of the bound"


CASES = [
    # T, Hq, Hkv, hd, rot, interleaved, scaling, norm
    (1, 12, 2, 128, None, False, YARN, False),
    (33, 4, 2, 64, None, False, LLAMA3, True),
    (5, 14, 2, 64, 32, True, LINEAR, False),
    (257, 3, 1, 128, 96, True, None, True),
    (2, 1, 1, 8, None, True, YARN, True),
    (19, 2, 2, 80, 40, False, LINEAR, True),
    (7, 4, 1, 256, 64, False, YARN, True),
    (1000, 16, 8, 128, 32, False, LLAMA3, False),
    (6001, 4, 2, 128, None, False, YARN, True),
    (3000, 32, 8, 128, None, False, None, False),
    (40, 5, 5, 72, 72, True, None, False),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_gradients(case):
    from meshy_b200.ops import reference as ref
    from meshy_b200.ops.rotary import qkv_rotary

    T, Hq, Hkv, hd, rot, inter, scaling, norm = case
    rope = _rope(hd, rot, inter, scaling)
    qkv, pos, qn, kn = _inputs(T, Hq, Hkv, hd, norm)
    gen = torch.Generator(device="cuda").manual_seed(7)
    grads = [torch.randn(T, n, hd, generator=gen, device="cuda").bfloat16() for n in (Hq, Hkv, Hkv)]

    leaves = [x.detach().clone().requires_grad_() for x in (qkv, qn, kn) if x is not None]
    out = qkv_rotary(leaves[0], pos, rope, Hq, Hkv, *(leaves[1:] or (None, None)), 1e-6)
    back = torch.autograd.grad(out, leaves, grads)

    exact = [x.detach().double().requires_grad_() for x in leaves]
    want = ref.qkv_rotary(exact[0], pos, rope, Hq, Hkv, *(exact[1:] or (None, None)), 1e-6)
    want_back = torch.autograd.grad(want, exact, [g.double() for g in grads])

    # In fp32: the angle to 2^-31 of a turn and its sine and cosine, three operations per pair (2^-21 of the pair's
    # size in all); with norms a sum of hd squares and a reciprocal root before (hd 2^-24 + 2^-21 of it).
    fine = 2.0 ** -21 + (hd * 2.0 ** -24 + 2.0 ** -21 if norm else 0.0)
    x = qkv.double().view(T, -1, hd)
    rstd = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)
    for i, (sl, w) in enumerate(((slice(0, Hq), qn), (slice(Hq, Hq + Hkv), kn))):
        y = x[:, sl] * rstd[:, sl] * w.double() if norm else x[:, sl]
        _near(out[i], want[i], fine * _size(y, rope))
    assert torch.equal(out[2], qkv.view(T, -1, hd)[:, Hq + Hkv:])
    assert torch.equal(back[0].view(T, -1, hd)[:, Hq + Hkv:], grads[2])
    gx, gx_want = back[0].view(T, -1, hd), want_back[0].view(T, -1, hd)
    for sl, w, g, j in ((slice(0, Hq), qn, grads[0], 1), (slice(Hq, Hq + Hkv), kn, grads[1], 2)):
        size = _size(g.double(), rope)  # of the gradient turned back
        if norm:
            u = (x * rstd)[:, sl].abs()
            d = size * w.double().abs()
            extra = 4 * fine * rstd[:, sl] * (d + u * (d * u).mean(-1, keepdim=True))
            # fp32 sums of T heads terms, each exact to ``fine``
            terms = (size * u).sum((0, 1))
            _near(back[j], want_back[j], (fine + 2.0 ** -24 * (T * g.shape[1] / 100 + 100)) * terms)
        else:
            extra = fine * size
        _near(gx[:, sl], gx_want[:, sl], extra)


def test_gradient_against_differences():
    """The gradient times a direction is the slope of the 64-bit definition along it."""
    from meshy_b200.ops import reference as ref
    from meshy_b200.ops.rotary import qkv_rotary

    T, Hq, Hkv, hd = 9, 4, 2, 64
    rope = _rope(hd, 48, True, YARN)
    qkv, pos, qn, kn = _inputs(T, Hq, Hkv, hd, True, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(5)
    grads = [torch.randn(T, n, hd, generator=gen, device="cuda").bfloat16() for n in (Hq, Hkv, Hkv)]
    leaves = [x.detach().clone().requires_grad_() for x in (qkv, qn, kn)]
    back = torch.autograd.grad(qkv_rotary(leaves[0], pos, rope, Hq, Hkv, *leaves[1:], 1e-6), leaves, grads)

    def value(args):
        out = ref.qkv_rotary(args[0], pos, rope, Hq, Hkv, *args[1:], 1e-6)
        return sum((o * g.double()).sum() for o, g in zip(out, grads))

    at = [x.double() for x in (qkv, qn, kn)]
    h = 2.0 ** -16
    for j in range(3):
        for _ in range(3):
            u = torch.randn(at[j].shape, generator=gen, device="cuda", dtype=torch.float64)
            step = [a + h * u if i == j else a for i, a in enumerate(at)]
            less = [a - h * u if i == j else a for i, a in enumerate(at)]
            slope = (value(step) - value(less)) / (2 * h)
            # each gradient entry is rounded to bf16; differences are exact to h^2 of the third derivative
            bound = 1.01 * BF16 * (back[j].double() * u).abs().sum() + 1e-4 * (1 + slope.abs())
            assert abs((back[j].double() * u).sum() - slope) <= bound


@pytest.mark.parametrize("inter", [False, True])
def test_far_positions(inter):
    """Angles stay exact where fp32 has none of the fraction left, to the last int32 position and below zero."""
    from meshy_b200.ops import reference as ref
    from meshy_b200.ops.rotary import qkv_rotary

    pos = torch.tensor([0, 1, -1, 131071, 131072, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, -(1 << 31)], dtype=torch.int32,
                       device="cuda")
    rope = _rope(128, None, inter, None, 5e5)
    qkv = _inputs(len(pos), 2, 1, 128, False)[0]
    out = qkv_rotary(qkv, pos, rope, 2, 1)
    want = ref.qkv_rotary(qkv.double(), pos, rope, 2, 1)
    # 2^31 radians in fp64 carry 2^-22 each, the table's turns 2^-33
    for o, w in zip(out[:2], want[:2]):
        _near(o, w, 2.0 ** -20 * 8)


def test_strided_and_empty_inputs():
    from meshy_b200.ops.rotary import qkv_rotary

    rope = _rope(64)
    wide = torch.randn(40, 1000, device="cuda").bfloat16()
    pos = torch.arange(40, dtype=torch.int32, device="cuda")
    plain = qkv_rotary(wide[:, 100:612].contiguous(), pos, rope, 4, 2)
    for view in (wide[:, 100:612], wide[:, 101:613], torch.stack((wide, wide), -1)[:, 100:612, 0]):
        same = wide[:, 101:613].contiguous() if view.data_ptr() == wide[:, 101:613].data_ptr() else None
        got = qkv_rotary(view, pos, rope, 4, 2)
        ref_out = plain if same is None else qkv_rotary(same, pos, rope, 4, 2)
        assert all(torch.equal(a, b) for a, b in zip(got, ref_out))
    none = qkv_rotary(wide[:0, :512], pos[:0], rope, 4, 2)
    assert [x.shape[0] for x in none] == [0, 0, 0]
    x = wide[:0, :512].detach().requires_grad_()
    w = torch.ones(64, device="cuda").bfloat16().requires_grad_()
    y = qkv_rotary(x, pos[:0], rope, 4, 2, w, w, 1e-6)
    g = torch.autograd.grad(y[0].sum(), (x, w))
    assert g[0].shape == x.shape and float(g[1].abs().sum()) == 0.0
    # a gradient that is broadcast, and outputs that nothing uses
    x = wide[:, :512].contiguous().requires_grad_()
    g1 = torch.autograd.grad(qkv_rotary(x, pos, rope, 4, 2)[0].float().sum(), x)[0]
    g2 = torch.autograd.grad(qkv_rotary(x, pos, rope, 4, 2), x, (torch.ones(40, 4, 64, device="cuda").bfloat16(),) + tuple(
        torch.zeros(40, 2, 64, device="cuda").bfloat16() for _ in "kv"))[0]
    assert torch.equal(g1, g2)


def test_main_grad_and_repeatable_sums():
    from meshy_b200.ops.rotary import qkv_rotary

    T, Hq, Hkv, hd = 3001, 8, 2, 128
    rope = _rope(hd, None, False, YARN)
    qkv, pos, qn, kn = _inputs(T, Hq, Hkv, hd, True)
    qn, kn = qn.requires_grad_(), kn.requires_grad_()
    g = [torch.randn(T, n, hd, device="cuda").bfloat16() for n in (Hq, Hkv, Hkv)]
    plain = torch.autograd.grad(qkv_rotary(qkv, pos, rope, Hq, Hkv, qn, kn), (qn, kn), g)
    sums = []
    for _ in range(2):
        for w in (qn, kn):
            w.main_grad = torch.full((hd,), 2.0, device="cuda")
        torch.autograd.backward(qkv_rotary(qkv.detach().requires_grad_(), pos, rope, Hq, Hkv, qn, kn), g)
        assert qn.grad is None and kn.grad is None
        sums.append([w.main_grad for w in (qn, kn)])
    for i in range(2):
        assert torch.equal(sums[0][i], sums[1][i])
        # 2 + g rounded to fp32 against g rounded to bf16
        _near(plain[i], sums[0][i].double() - 2.0, 2.0 ** -23 * (2 + sums[0][i].double().abs()))


def test_frozen_norms_and_second_derivatives():
    from meshy_b200.ops.rotary import qkv_rotary

    rope = _rope(64)
    qkv, pos, qn, kn = _inputs(5, 2, 1, 64, True)
    qn.main_grad = torch.zeros(64, device="cuda")  # frozen: nothing is added
    kn.requires_grad_()
    kn.main_grad = torch.zeros(64, device="cuda")
    x = qkv.detach().requires_grad_()
    out = qkv_rotary(x, pos, rope, 2, 1, qn, kn)
    torch.autograd.backward(out, [torch.ones_like(o) for o in out])
    assert float(qn.main_grad.abs().sum()) == 0.0 and float(kn.main_grad.abs().sum()) > 0.0 and x.grad is not None
    out = qkv_rotary(x, pos, rope, 2, 1)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(out[0].float().pow(2).sum(), x, create_graph=True)
    with torch.inference_mode():
        a = qkv_rotary(qkv, pos, _rope(64, 32, False, LINEAR, 7e4), 2, 1)
    b = qkv_rotary(x, pos, _rope(64, 32, False, LINEAR, 7e4), 2, 1)
    assert torch.equal(a[0], b[0])
    torch.autograd.grad(b[0].float().sum(), x)


def test_activation_checkpoint_and_retained_graph():
    from torch.utils.checkpoint import checkpoint

    from meshy_b200.ops.rotary import qkv_rotary

    rope = _rope(64, 32, True, YARN)
    qkv, pos, qn, kn = _inputs(70, 4, 2, 64, True)
    leaves = [x.requires_grad_() for x in (qkv, qn, kn)]
    g = [torch.randn(70, n, 64, device="cuda").bfloat16() for n in (4, 2, 2)]
    want = torch.autograd.grad(qkv_rotary(qkv, pos, rope, 4, 2, qn, kn), leaves, g)
    out = checkpoint(lambda x, a, b: qkv_rotary(x * 1.0, pos, rope, 4, 2, a, b), *leaves, use_reentrant=False)
    got = torch.autograd.grad(out, leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    out = qkv_rotary(qkv, pos, rope, 4, 2, qn, kn)
    for _ in range(2):
        got = torch.autograd.grad(out, leaves, g, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_projection_is_kept_for_the_norms_alone():
    """Without norms the gradient does not read the projection: it is not held, and may be written to in between."""
    from meshy_b200.ops.rotary import qkv_rotary

    rope = _rope(64)
    for norm in (False, True):
        qkv, pos, qn, kn = _inputs(100, 4, 2, 64, norm)
        leaf = qkv.clone().requires_grad_()
        x = leaf * 1
        out = qkv_rotary(x, pos, rope, 4, 2, qn, kn)
        grads = [torch.randn_like(o) for o in out]
        want = torch.autograd.grad(out, leaf, grads, retain_graph=True)[0]
        with torch.no_grad():
            x.zero_()
        if norm:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(out, leaf, grads)
        else:
            assert torch.equal(torch.autograd.grad(out, leaf, grads)[0], want)


def test_cache_destination():
    from meshy_b200.ops.rotary import qkv_rotary, qkv_rotary_to_cache

    T, Hq, Hkv, hd, page = 37, 4, 2, 128, 16
    rope = _rope(hd, 64, True, LINEAR)
    qkv, pos, _, _ = _inputs(T, Hq, Hkv, hd, False)
    q, k, v = qkv_rotary(qkv, pos, rope, Hq, Hkv)
    kc, vc = (torch.full((6, Hkv, page, hd), 3.0, device="cuda").bfloat16() for _ in "kv")
    slots = torch.randperm(6 * page, device="cuda")[:T]
    slots[5], slots[6], slots[7] = -1, 6 * page, 1 << 40
    for keep in (False, True):
        a, b, c = (x.clone() for x in (kc, vc, slots))
        got = qkv_rotary_to_cache(qkv, pos, rope, Hq, Hkv, None, None, 1e-6, a, b, c, keep_kv=keep)
        assert torch.equal(got[0], q) and (got[1] is None) == (not keep)
        if keep:
            assert torch.equal(got[1], k) and torch.equal(got[2], v)
        want_k, want_v = kc.clone(), vc.clone()
        ok = (slots >= 0) & (slots < 6 * page)
        want_k[slots[ok] // page, :, slots[ok] % page] = k[ok]
        want_v[slots[ok] // page, :, slots[ok] % page] = v[ok]
        assert torch.equal(a, want_k) and torch.equal(b, want_v)


def test_capture_and_streams():
    from meshy_b200.ops.rotary import qkv_rotary

    T, Hq, Hkv, hd = 65, 4, 2, 64
    rope = _rope(hd, None, True, LLAMA3)
    qkv, pos, qn, kn = _inputs(T, Hq, Hkv, hd, True)
    qkv, qn, kn = (x.requires_grad_() for x in (qkv, qn, kn))
    g = [torch.randn(T, n, hd, device="cuda").bfloat16() for n in (Hq, Hkv, Hkv)]

    def step():
        out = qkv_rotary(qkv, pos, rope, Hq, Hkv, qn, kn)
        return (*out, *torch.autograd.grad(out, (qkv, qn, kn), g))

    fresh = _rope(hd, 16, False, YARN, 1e6)
    with pytest.raises(RuntimeError, match="before a CUDA graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            qkv_rotary(qkv.detach(), pos, fresh, Hq, Hkv)
    want = [x.detach().clone() for x in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    del other
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        pos.add_(11)
    graph.replay()
    again = [x.detach().clone() for x in held]
    del held
    assert all(torch.equal(a, b) for a, b in zip(again, step()))
    assert not torch.equal(again[0], want[0])


@pytest.mark.parametrize("norm", [False, True])
def test_rows_beyond_32_bits(norm):
    """More than 2^31 channels in one call: its last rows hold what a call on them alone gives."""
    from meshy_b200.ops.rotary import qkv_rotary

    T, Hq, Hkv, hd, n = (1 << 20) + 640, 4, 2, 256, 1000
    rope = _rope(hd, 64, norm, YARN)
    qkv, pos, qn, kn = _inputs(n, Hq, Hkv, hd, norm)
    at = torch.arange(T, device="cuda") % n
    x, p = qkv[at].requires_grad_(), pos[at]
    out = qkv_rotary(x, p, rope, Hq, Hkv, qn, kn)
    grads = [g.contiguous() for g in (o.detach().flip(-1) for o in out)]
    dx = torch.autograd.grad(out, x, grads)[0]
    few = x.detach()[-n:].clone().requires_grad_()
    want = qkv_rotary(few, p[-n:], rope, Hq, Hkv, qn, kn)
    dw = torch.autograd.grad(want, few, [g[-n:] for g in grads])[0]
    assert all(torch.equal(a[-n:], b) for a, b in zip(out, want)) and torch.equal(dx[-n:], dw)


def test_refusals():
    from meshy_b200.ops._ext import ext
    from meshy_b200.ops.rotary import qkv_rotary, qkv_rotary_to_cache

    rope = _rope(64)
    qkv, pos, qn, kn = _inputs(4, 2, 1, 64, True)
    for args in ((qkv[:, :-1], pos, rope, 2, 1), (qkv, pos.long(), rope, 2, 1), (qkv, pos[:3], rope, 2, 1),
                 (qkv, pos, rope, 2, 1, qn, None), (qkv, pos, rope, 0, 1), (qkv[0], pos, rope, 2, 1)):
        with pytest.raises(ValueError):
            qkv_rotary(*args)
    for args in ((qkv.float(), pos, rope, 2, 1), (qkv, pos.cpu(), rope, 2, 1), (qkv, pos, rope, 2, 1, qn.float(), kn.float()),
                 (qkv, pos, rope, 2, 1, qn[:32], kn[:32])):
        with pytest.raises(RuntimeError):
            qkv_rotary(*args)
    kc = torch.zeros(2, 1, 16, 64, device="cuda").bfloat16()
    slots = torch.arange(4, device="cuda")
    for k, v, s in ((kc, kc[:1], slots), (kc.float(), kc.float(), slots), (kc, kc, slots.int()), (kc, kc, slots[:3])):
        with pytest.raises(RuntimeError):
            qkv_rotary_to_cache(qkv, pos, rope, 2, 1, None, None, 1e-6, k, v, s)
    with pytest.raises(RuntimeError):  # a table for another width
        ext().rotary_fwd(qkv, pos, torch.zeros(64, dtype=torch.int64, device="cuda"), 1.0, False, None, None, 2, 1, 64, 1e-6,
                         None, None, None, True)
