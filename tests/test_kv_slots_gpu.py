"""Rows without a slot (below zero) are not written to the paged cache, whichever kernel writes it (GPU). The caches lie
between guards that nothing may touch."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _bf(*shape):
    return torch.randn(*shape, device=DEV).bfloat16()


def _caches(pages, Hkv, page, hd):
    """K and V with a page of guard before, between and behind them; the whole buffer."""
    n = Hkv * page * hd
    raw = torch.full(((2 * pages + 3) * n,), 7.0, dtype=torch.bfloat16, device=DEV)
    at = [raw[n * (1 + i * (pages + 1)):][:pages * n].view(pages, Hkv, page, hd) for i in range(2)]
    return raw, at[0], at[1]


def _want(raw, k, v, slots, pages, Hkv, page, hd):
    want = torch.full_like(raw, 7.0)
    n = Hkv * page * hd
    for i, x in enumerate((k, v)):
        cache = want[n * (1 + i * (pages + 1)):][:pages * n].view(pages, Hkv, page, hd)
        for t, s in enumerate(slots.tolist()):
            if s >= 0:
                cache[s // page, :, s % page] = x[t]
    return want


SLOTS = [191, -1, 0, -64, 70, -1, 64, -(1 << 40)]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("norm", [False, True])
def test_plain_rope_and_scatter(hd, norm):
    from meshy_b200.ops import decode as D

    torch.manual_seed(1)
    T, Hq, Hkv, pages, page = len(SLOTS), 4, 2, 3, 64
    qkv, pos = _bf(T, (Hq + 2 * Hkv) * hd), torch.arange(T, dtype=torch.int32, device=DEV)
    w = (_bf(hd), _bf(hd)) if norm else (None, None)
    slots = torch.tensor(SLOTS, device=DEV)
    raw, kc, vc = _caches(pages, Hkv, page, hd)
    _, k, v = D.qkv_rope_to_cache(qkv, pos, *w, Hq, Hkv, hd, 1e4, 1e-6, kc, vc, slots, keep_kv=True)
    assert torch.equal(raw, _want(raw, k, v, slots, pages, Hkv, page, hd))
    raw, kc, vc = _caches(pages, Hkv, page, hd)
    D.kv_write(k, v, kc, vc, slots)
    assert torch.equal(raw, _want(raw, k, v, slots, pages, Hkv, page, hd))


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("T", [1, 8, 33])
def test_fused_projection(T, norm):
    from meshy_b200.ops import decode as D

    torch.manual_seed(2)
    Hq, Hkv, hd, pages, page, dim = 4, 2, 128, 3, 64, 512
    x, wt, pos = _bf(T, dim), _bf((Hq + 2 * Hkv) * hd, dim) * 0.05, torch.arange(T, dtype=torch.int32, device=DEV)
    w = (_bf(hd), _bf(hd)) if norm else (None, None)
    slots = torch.tensor([s if i % 3 else -1 for i, s in enumerate(torch.randperm(pages * page)[:T].tolist())], device=DEV)
    full = torch.arange(T, device=DEV)
    raw0, kc0, vc0 = _caches(pages, Hkv, page, hd)
    q0 = D.qkv_rope_fused(x, wt, None, pos, *w, Hq, Hkv, 1e4, 1e-6, kc0, vc0, full)
    assert q0 is not None
    k, v = (c.transpose(1, 2).reshape(-1, Hkv, hd)[:T] for c in (kc0, vc0))
    raw, kc, vc = _caches(pages, Hkv, page, hd)
    q = D.qkv_rope_fused(x, wt, None, pos, *w, Hq, Hkv, 1e4, 1e-6, kc, vc, slots)
    assert torch.equal(q, q0) and torch.equal(raw, _want(raw, k, v, slots, pages, Hkv, page, hd))


def test_whole_step_kernel(monkeypatch):
    """One row of three without a slot: the cache changes where the per-kernel path changes it, nowhere else."""
    from meshy_b200.models.args import ModelArgs
    from meshy_b200.ops._ext import ext
    from meshy_b200.rollout import RolloutEngine

    monkeypatch.setenv("MESHY_MEGA", "1")
    args = ModelArgs(name="qwen2_5", flavor="slots_test", dim=512, n_layers=3, n_heads=8, n_kv_heads=2, head_dim=128,
                     ffn_dim=1024, vocab_size=4096, rope_theta=1e6, qkv_bias=True, max_seq_len=1024)
    e = RolloutEngine(args, device=DEV, max_running=8, max_total_tokens=4096, page_size=64, max_seq_len=1024,
                      use_cuda_graph=False, seed=0)
    assert e._mega is not None, e.mega_reason
    for n in (5, 70, 130):
        e.submit([3 + i % 1000 for i in range(n)], 16, ignore_eos=True)
    e._admit()
    e._ensure_pages(range(3), 2)
    e.st["slot"][1] = -1
    before = e.kv.clone()
    want = e._decode_hidden_layers(3).clone()
    after = e.kv.clone()
    e.kv.copy_(before)
    ext().clear_device_error()
    got = e._mega(e.st, 3).clone()
    torch.cuda.synchronize()
    assert int(ext().device_error()) == 0
    rows = (after != before).any(-1)
    assert rows.any() and torch.equal((e.kv != before).any(-1), rows)
    # two rows of three layers, two KV heads, K and V
    assert int(rows.sum()) == 2 * 3 * 2 * 2
    assert ((got.float() - want.float()).norm() / want.float().norm()).item() < 2e-2  # as bf16 steps in another order give
