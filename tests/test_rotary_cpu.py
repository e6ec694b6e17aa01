"""Rotary positions in any layout and scaling on the CPU: frequencies, gradients, model configurations, refusals."""

import dataclasses
import json
import math

import pytest
import torch

from meshy_b200.models import build_model, get_model_args, with_hf_config
from meshy_b200.models.hf import from_hf, hf_config
from meshy_b200.ops.rotary import Rope, RopeScaling, make_rope, qkv_rotary, qkv_rotary_to_cache

YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 64}
LINEAR = {"type": "linear", "factor": 2.5}


def test_plain_frequencies_and_turns():
    r = Rope(64, 5e5)
    f = r.frequencies()
    assert f == [5e5 ** (-i / 32) for i in range(32)] and r.factor == 1.0
    turns = r.turns("cpu")
    assert turns is r.turns("cpu") and turns.dtype == torch.int64
    for i in (0, 5, 31):
        got = (int(turns[i]) % (1 << 64)) / 2.0 ** 64
        assert got == pytest.approx(f[i] / (2 * math.pi), rel=1e-15)
    # a whole number of positions wraps exactly: 2^20 times the fraction, modulo one
    assert ((int(turns[0]) << 20) % (1 << 64)) / 2.0 ** 64 == pytest.approx((2 ** 20 / (2 * math.pi)) % 1.0, abs=1e-9)


def test_scaled_frequencies():
    base = Rope(64, 1e4).frequencies()
    assert Rope(64, 1e4, scaling=LINEAR).frequencies() == [x / 2.5 for x in base]
    got = Rope(64, 1e4, scaling=LLAMA3).frequencies()
    for x, y in zip(base, got):
        length = 2 * math.pi / x
        if length < 64 / 4:
            assert y == pytest.approx(x, rel=1e-15)
        elif length > 64:
            assert y == pytest.approx(x / 8, rel=1e-15)
        else:
            mix = (64 / length - 1) / 3
            assert y == pytest.approx((1 - mix) * x / 8 + mix * x, rel=1e-12)
    r = Rope(64, 1e4, scaling=YARN)
    assert r.factor == pytest.approx(0.1 * math.log(4.0) + 1)
    at = lambda turns: 64 * math.log(64 / (turns * 2 * math.pi)) / (2 * math.log(1e4))  # noqa: E731
    lo, hi = max(math.floor(at(32)), 0), min(math.ceil(at(1)), 63)
    for i, (x, y) in enumerate(zip(base, r.frequencies())):
        ramp = min(max((i - lo) / (hi - lo), 0), 1)
        assert y == pytest.approx(x / 4 * ramp + x * (1 - ramp), rel=1e-12)
    assert Rope(64, scaling={**YARN, "attention_factor": 2.0}).factor == 2.0
    assert Rope(64, scaling={"rope_type": "default"}).scaling is None


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("rot", [8, 16])
@pytest.mark.parametrize("norm", [False, True])
def test_gradients_against_differences(inter, rot, norm):
    rope = Rope(16, 100.0, rot, inter, YARN)
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(3, (2 + 2) * 16, generator=g, dtype=torch.float64, requires_grad=True)
    pos = torch.tensor([0, 7, 100000], dtype=torch.int32)
    ws = [torch.randn(16, generator=g, dtype=torch.float64, requires_grad=True) for _ in "qk"] if norm else []
    f = lambda x, *w: qkv_rotary(x, pos, rope, 2, 1, *(w or (None, None)), 1e-6)  # noqa: E731
    assert torch.autograd.gradcheck(f, (qkv, *ws))


def test_layouts_are_permutations_of_each_other():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 3 * 32, generator=g)
    pos = torch.randint(0, 1000, (5,), generator=g).int()
    order = torch.arange(16).view(2, 8).t().reshape(-1)  # halves -> neighbours
    a = qkv_rotary(x, pos, Rope(32, rotary_dim=16), 1, 1)
    swapped = x.view(5, 3, 32).clone()
    swapped[..., :16] = swapped[..., :16][..., order]
    b = qkv_rotary(swapped.view(5, -1), pos, Rope(32, rotary_dim=16, interleaved=True), 1, 1)
    for y, z in zip(a[:2], b[:2]):
        assert torch.allclose(y[..., :16][..., order], z[..., :16], atol=1e-6) and torch.equal(y[..., 16:], z[..., 16:])
    assert torch.equal(a[0][..., 16:], x.view(5, 3, 32)[:, :1, 16:])


def test_cache_destination_skips_slots_outside():
    x = torch.randn(4, 3 * 32)
    pos = torch.arange(4, dtype=torch.int32)
    rope = Rope(32, interleaved=True)
    kc, vc = torch.zeros(2, 1, 4, 32), torch.zeros(2, 1, 4, 32)
    q, k, v = qkv_rotary(x, pos, rope, 1, 1)
    got = qkv_rotary_to_cache(x, pos, rope, 1, 1, None, None, 1e-6, kc, vc, torch.tensor([5, -1, 8, 0]), keep_kv=True)
    assert all(torch.equal(a, b) for a, b in zip(got, (q, k, v)))
    assert torch.equal(kc[1, 0, 1], k[0, 0]) and torch.equal(vc[0, 0, 0], v[3, 0]) and int((kc != 0).any(-1).sum()) == 2


@pytest.mark.parametrize("bad", [
    dict(head_dim=12), dict(head_dim=0), dict(head_dim=264), dict(head_dim=64, rotary_dim=12), dict(head_dim=64, rotary_dim=72),
    dict(head_dim=64, rotary_dim=0), dict(head_dim=64, theta=1.0), dict(head_dim=64, theta=math.inf),
    dict(head_dim=64, scaling={"rope_type": "dynamic", "factor": 2.0}), dict(head_dim=64, scaling={"rope_type": "yarn", "factor": 2.0}),
    dict(head_dim=64, scaling={"rope_type": "linear"}), dict(head_dim=64, scaling={"rope_type": "linear", "factor": 0.5}),
    dict(head_dim=64, scaling={**LLAMA3, "low_freq_factor": 4.0}), dict(head_dim=64, scaling={**YARN, "mscale": 1.0}),
    dict(head_dim=64, scaling={**YARN, "beta_fast": 1.0}), dict(head_dim=64, scaling={**YARN, "attention_factor": 0.0}),
    dict(head_dim=64, scaling={"rope_type": "linear", "factor": math.nan}),
], ids=str)
def test_refused_configurations(bad):
    with pytest.raises(ValueError):
        Rope(**bad)


def test_refused_calls():
    r, x, p = Rope(32), torch.randn(4, 96), torch.arange(4, dtype=torch.int32)
    for args in ((x[:, 1:], p, r, 1, 1), (x, p.long(), r, 1, 1), (x, p[1:], r, 1, 1), (x, p, r, 1, 1, torch.ones(32), None),
                 (x[None], p, r, 1, 1)):
        with pytest.raises(ValueError):
            qkv_rotary(*args)


def test_model_configuration():
    a = get_model_args("llama3", "debugmodel")
    assert a.rope is None and with_hf_config(a, None) is a
    b = with_hf_config(a, {"rope_scaling": LLAMA3, "rope_theta": 1e6, "max_position_embeddings": 9999})
    assert b.rope == Rope(64, 1e6, scaling=LLAMA3) and b.rope is b.rope and b.max_seq_len == 9999 and hash(b) == hash(b)
    c = with_hf_config(a, {"rope_parameters": {**YARN, "rope_theta": 2e4}, "partial_rotary_factor": 0.5, "rope_interleaved": True})
    assert c.rope == Rope(64, 2e4, 32, True, YARN) and c.rope is make_rope(64, 2e4, 32, True, RopeScaling.of(YARN))
    for args in (b, c, a):  # what is exported is what is read
        cfg = json.loads(json.dumps(hf_config(args)))
        back = with_hf_config(a, {k: cfg[k] for k in ("rope_theta", "rope_scaling", "partial_rotary_factor", "rope_interleaved",
                                                     "max_position_embeddings") if k in cfg})
        assert back == dataclasses.replace(args)
    assert get_model_args("llama3", "debugmodel", rope_scaling=LLAMA3).rope.scaling.factor == 8.0
    for bad in ({"rope_scale": 2}, {"rope_scaling": {"rope_type": "linear"}}, {"partial_rotary_factor": 0.3}):
        with pytest.raises(ValueError):
            with_hf_config(a, bad)
    with pytest.raises(ValueError, match="unknown model fields"):
        get_model_args("llama3", "debugmodel", rope_scalling=LLAMA3)


def test_exported_part_of_a_head_is_read_back():
    """The factor times the head's width is cut off to a whole number, by this reader and others."""
    a = get_model_args("llama3", "debugmodel")
    for hd in range(8, 257, 8):
        for rot in range(8, hd, 8):
            args = dataclasses.replace(a, head_dim=hd, rope_dim=rot)
            cfg = hf_config(args)
            back = with_hf_config(dataclasses.replace(args, rope_dim=None),
                                  {"partial_rotary_factor": json.loads(json.dumps(cfg["partial_rotary_factor"]))})
            assert back.rope_dim == rot, (hd, rot)


@pytest.mark.parametrize("scaling", [LLAMA3, YARN, LINEAR], ids=lambda s: s.get("rope_type", "linear"))
def test_logits_match_hf_llama_with_scaling(scaling):
    from transformers import LlamaConfig, LlamaForCausalLM

    a = get_model_args("llama3", "debugmodel", vocab_size=512, rope_theta=1e4, rope_scaling=scaling)
    hf_scaling = {("rope_type" if k == "type" else k): v for k, v in scaling.items()}
    cfg = LlamaConfig(hidden_size=a.dim, num_hidden_layers=a.n_layers, num_attention_heads=a.n_heads,
                      num_key_value_heads=a.n_kv_heads, head_dim=a.head_dim, intermediate_size=a.ffn_dim,
                      vocab_size=a.vocab_size, rms_norm_eps=a.norm_eps, tie_word_embeddings=False,
                      max_position_embeddings=256, attention_bias=False, mlp_bias=False,
                      rope_parameters={"rope_theta": a.rope_theta, **hf_scaling})
    torch.manual_seed(0)
    hf = LlamaForCausalLM(cfg).float().eval()
    ours = build_model(a, seed=1, device="cpu", dtype=torch.float32).eval()
    sd = from_hf(a, dict(hf.state_dict()))
    with torch.no_grad():
        for name, p in ours.named_parameters():
            p.copy_(sd[name])
        ids = torch.randint(0, a.vocab_size, (1, 150))
        want = hf(input_ids=ids).logits[0]
        got = ours.logits(ids[0], torch.arange(150, dtype=torch.int32), torch.tensor([0, 150], dtype=torch.int32), 150)
    assert torch.allclose(got.float(), want, atol=2e-4, rtol=1e-4), (got - want).abs().max()


def test_trainer_takes_the_overrides():
    from meshy_b200.backend.trainer import PPOTrainer
    from meshy_b200.config import TrainerConfig, TrainerParamsConfig

    tc = TrainerConfig(model_name="qwen3", model_flavor="debugmodel", seq_len=64,
                       model_overrides={"rope_scaling": YARN, "partial_rotary_factor": 0.5})
    t = PPOTrainer(tc, TrainerParamsConfig(mini_batch_size=2), device="cpu")
    assert t.model_args.rope == Rope(64, 1e6, 32, False, YARN)
