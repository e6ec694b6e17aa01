"""Rollout engine with an 8-bit KV cache and scaled rotary positions on the GPU: captured steps against eager ones,
the engine's log-probs against the model's."""

import pytest
import torch

pytestmark = pytest.mark.gpu

PROMPTS = [[5, 9, 77, 300, 12], [1, 2, 3], list(range(40, 175)), [7] * 64]
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 128}
ROPES = [{}, {"rope_scaling": YARN}, {"partial_rotary_factor": 0.5, "rope_interleaved": True}]


def _engine(flavor=("qwen3", "debugmodel"), overrides=None, fields=None, **kw):
    from meshy_b200.models import build_model, get_model_args, with_hf_config
    from meshy_b200.rollout.engine import RolloutEngine

    args = with_hf_config(get_model_args(*flavor, **(fields or {})), overrides)
    model = build_model(args, seed=3, device="cuda", dtype=torch.bfloat16)
    return RolloutEngine(args, device="cuda", model=model, max_running=8, max_total_tokens=8192, max_seq_len=512, sync_every=4, **kw)


@pytest.mark.parametrize("kv_dtype", ["auto", "int8"])
@pytest.mark.parametrize("rope", ROPES, ids=["plain", "yarn", "part"])
@pytest.mark.parametrize("sampling", [dict(temperature=0.0), dict(temperature=0.8)])
def test_captured_steps_match_eager_ones(kv_dtype, rope, sampling):
    a = _engine(overrides=rope, kv_dtype=kv_dtype).generate(PROMPTS, 21, **sampling)
    b = _engine(overrides=rope, kv_dtype=kv_dtype, use_cuda_graph=False).generate(PROMPTS, 21, **sampling)
    for x, y in zip(a, b):
        assert x.output_ids == y.output_ids
        assert x.output_logprobs == pytest.approx(y.output_logprobs, abs=2e-2)


@pytest.mark.parametrize("kv_dtype", ["auto", "int8"])
@pytest.mark.parametrize("rope", ROPES, ids=["plain", "yarn", "part"])
def test_engine_and_model_agree(kv_dtype, rope):
    """Log-probs of the drawn tokens in the engine and in the training forward (bf16 sums in another order; 8-bit keys and
    values are off by a 254th of their block's largest: 0.06 at logits of unit spread)."""
    e = _engine(overrides=rope, kv_dtype=kv_dtype)
    g = e.generate([list(range(40, 175))], 40, temperature=1.0, ignore_eos=True)[0]
    ids = torch.tensor(g.tokens, device="cuda")
    n, p = len(ids), len(g.prompt_ids)
    with torch.no_grad():
        logits = e.model.logits(ids, torch.arange(n, dtype=torch.int32, device="cuda"),
                                torch.tensor([0, n], dtype=torch.int32, device="cuda"), n)
    lp = torch.log_softmax(logits.float(), -1)[torch.arange(p - 1, n - 1), ids[p:]]
    assert torch.allclose(lp.cpu(), torch.tensor(g.output_logprobs), atol=6e-2)


def test_head_width_128_wide_groups_and_memory():
    fields = dict(n_layers=2, vocab_size=4096)
    e = _engine(("qwen2_5_math", "R1-Distill-1.5B"), fields=fields, kv_dtype="int8")
    full = _engine(("qwen2_5_math", "R1-Distill-1.5B"), fields=fields)
    a, b = (x.generate([[3, 1, 4] * 100, [2, 7] * 9], 40, temperature=0.0) for x in (e, full))
    assert all(len(g.output_ids) == 40 for g in a + b)
    assert e._kv_bytes_per_token() / full._kv_bytes_per_token() == (16 * 256 + 8) / (16 * 512)
    assert e.mega_reason == "8-bit KV cache"


def test_release_and_resume_keep_the_captured_steps():
    e = _engine(kv_dtype="int8")
    want = [g.output_ids for g in e.generate(PROMPTS, 12, temperature=0.0)]
    at = e.kv[0].k.data_ptr()
    e.release_memory()
    with pytest.raises(RuntimeError, match="released"):
        e.generate(PROMPTS, 2)
    e.waiting.clear()
    e.resume_memory()
    assert e.kv[0].k.data_ptr() == at
    assert [g.output_ids for g in e.generate(PROMPTS, 12, temperature=0.0)] == want


def test_training_step_with_scaled_positions():
    """Gradients of the model's loss with partly rotated, scaled heads against fp32 autograd of the same model."""
    from meshy_b200.models import build_model, get_model_args, with_hf_config
    from meshy_b200.ops import functional as Fx

    args = with_hf_config(get_model_args("qwen3", "debugmodel"), {"rope_scaling": YARN, "partial_rotary_factor": 0.5})
    ours = build_model(args, seed=3, device="cuda", dtype=torch.bfloat16)
    full = build_model(args, seed=3, device="cuda", dtype=torch.bfloat16).float()
    ids = torch.randint(0, args.vocab_size, (200,), device="cuda")
    pos = torch.cat([torch.arange(120), torch.arange(80)]).int().cuda()
    cu = torch.tensor([0, 120, 200], dtype=torch.int32, device="cuda")
    labels = torch.roll(ids, -1)
    grads = []
    for m, base in ((ours, False), (full, True)):
        with Fx.torch_baseline(base):
            lp, _ = m.logprobs(ids, labels, pos, cu, 120)
            grads.append(torch.autograd.grad(lp.float().mean(), [m.layers[0].wqkv, m.layers[0].q_norm, m.layers[1].k_norm]))
    for a, b in zip(*grads):  # bf16 activations throughout: a few of their roundings (2^-8) in the norm of the difference
        assert float((a.float() - b).norm() / b.norm()) < 0.05
