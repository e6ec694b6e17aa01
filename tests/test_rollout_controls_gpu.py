"""Rollout engine with a 4-bit KV cache and with logit controls on the GPU: captured decode steps against eager ones."""

import pytest
import torch

pytestmark = pytest.mark.gpu

PROMPTS = [[5, 9, 77, 300, 12], [1, 2, 3], list(range(40, 175)), [7] * 64]


def _engine(flavor=("qwen3", "debugmodel"), **kw):
    from meshy_b200.models import build_model, get_model_args
    from meshy_b200.rollout.engine import RolloutEngine

    args = get_model_args(*flavor)
    model = build_model(args, seed=3, device="cuda", dtype=torch.bfloat16)
    return RolloutEngine(args, device="cuda", model=model, max_running=8, max_total_tokens=8192, max_seq_len=512, sync_every=4, **kw)


CONTROLS = dict(repetition_penalty=1.3, frequency_penalty=0.2, presence_penalty=0.3, logit_bias={11: 2.0, 2047: -3.0},
                allowed_tokens=list(range(5, 1900)))


@pytest.mark.parametrize("kv_dtype", ["auto", "int4"])
@pytest.mark.parametrize("sampling", [dict(temperature=0.0), dict(temperature=0.8), dict(temperature=1.0, top_k=5, top_p=0.9)])
@pytest.mark.parametrize("controls", [{}, CONTROLS])
def test_captured_steps_match_eager_ones(kv_dtype, sampling, controls):
    a = _engine(kv_dtype=kv_dtype).generate(PROMPTS, 21, **sampling, **controls)
    b = _engine(kv_dtype=kv_dtype, use_cuda_graph=False).generate(PROMPTS, 21, **sampling, **controls)
    for x, y in zip(a, b):
        assert x.output_ids == y.output_ids
        assert x.output_logprobs == pytest.approx(y.output_logprobs, abs=2e-2)
        if controls:
            assert all(5 <= t < 1900 for t in x.output_ids)


def test_presence_penalty_counts_in_replayed_steps():
    e = _engine(kv_dtype="int4")
    for _ in range(2):  # the second call runs captured steps only, on reused slots
        out = [g.output_ids for g in e.generate(PROMPTS, 60, temperature=0.0, presence_penalty=1e4)]
        assert all(len(set(o)) == 60 for o in out)
    assert e.stats["graph_replays"] > 0


def test_plain_requests_beside_controlled_ones():
    plain = [g.output_ids for g in _engine().generate(PROMPTS, 24, temperature=0.0)]
    e = _engine()
    rids = [e.submit(p, 24, temperature=0.0, **(CONTROLS if i == 1 else {})) for i, p in enumerate(PROMPTS)]
    e.run_until_idle()
    got = [e.finished[r].output_ids for r in rids]
    assert [g for i, g in enumerate(got) if i != 1] == [p for i, p in enumerate(plain) if i != 1]
    assert all(5 <= t < 1900 for t in got[1])


def test_release_and_resume_keep_the_captured_steps():
    e = _engine(kv_dtype="int4")
    want = [g.output_ids for g in e.generate(PROMPTS, 12, temperature=0.0)]
    at = e.kv[0].k.data_ptr()
    e.release_memory()
    with pytest.raises(RuntimeError, match="released"):
        e.generate(PROMPTS, 2)
    e.waiting.clear()
    e.resume_memory()
    assert e.kv[0].k.data_ptr() == at
    assert [g.output_ids for g in e.generate(PROMPTS, 12, temperature=0.0)] == want


def test_head_width_128_and_bias_model():
    from meshy_b200.models import build_model, get_model_args
    from meshy_b200.rollout.engine import RolloutEngine

    args = get_model_args("qwen2_5_math", "R1-Distill-1.5B", n_layers=2, vocab_size=4096)
    model = build_model(args, seed=1, device="cuda", dtype=torch.bfloat16)
    out = []
    for kv in ("auto", "int4"):
        e = RolloutEngine(args, device="cuda", model=model, max_running=8, max_total_tokens=16384, max_seq_len=2048, kv_dtype=kv)
        out.append(e.generate([[3, 1, 4] * 100, [2, 7] * 9], 40, temperature=0.0))
    # a random model's next token is a near tie, so only the shapes and the first steps' agreement say something
    assert all(len(g.output_ids) == 40 for o in out for g in o)


def test_whole_step_kernel_is_off_for_the_4bit_cache_and_says_why():
    assert _engine(kv_dtype="int4").mega_reason == "4-bit KV cache"
    assert _engine().mega_reason is None or "4-bit" not in _engine().mega_reason


@pytest.mark.parametrize("flavor,kw", [(("qwen2_5_math", "R1-Distill-1.5B"), dict(n_layers=2, vocab_size=4096)),
                                       (("qwen3", "debugmodel"), {})])
def test_int4_prefill_and_decode_see_the_same_cache(flavor, kw):
    """A prompt that ends before a generated token gives that token the log-probability that it had when it was drawn:
    decode attends to the cache, prefill reads it back. (Log-probs differ by the order of bf16 sums and by keys that land
    on the other side of a nibble's step: 0.05 at logits of unit spread.)"""
    from meshy_b200.models import build_model, get_model_args
    from meshy_b200.rollout.engine import RolloutEngine

    args = get_model_args(*flavor, **kw)
    model = build_model(args, seed=1, device="cuda", dtype=torch.bfloat16)
    e = RolloutEngine(args, device="cuda", model=model, max_running=8, max_total_tokens=16384, max_seq_len=1024,
                      kv_dtype="int4", sync_every=4)
    g = e.generate([[3, 1, 4, 15] * 40], 24, temperature=1.0, ignore_eos=True)[0]
    seen, sample = [], e._sample_rows

    def spy(h, reqs):
        seen.append(torch.log_softmax(h.float() @ e.model.output_weight.float().t(), -1))
        return sample(h, reqs)

    e._sample_rows = spy
    for i, (tok, lp) in enumerate(zip(g.output_ids, g.output_logprobs)):
        e.generate([g.prompt_ids + g.output_ids[:i]], 1, temperature=1.0)
        assert float(seen[-1][0, tok]) == pytest.approx(lp, abs=5e-2), i
