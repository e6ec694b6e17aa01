"""Rollout engine with an 8-bit KV cache, device-made tables and scaled rotary positions, on the CPU."""

import pytest
import torch

from meshy_b200.models import build_model, get_model_args, with_hf_config
from meshy_b200.rollout.engine import RolloutEngine

PROMPTS = [[5, 9, 77, 300, 12], [1, 2, 3], list(range(40, 75)), [7] * 33]
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}


def _engine(overrides=None, **kw):
    args = with_hf_config(get_model_args("qwen3", "debugmodel"), overrides)
    model = build_model(args, seed=3)
    return RolloutEngine(args, model=model, max_running=4, max_total_tokens=2048, max_seq_len=256, page_size=16,
                         sync_every=3, **kw)


def _greedy(e, prompts, n, **kw):
    return [g.output_ids for g in e.generate(prompts, n, temperature=0.0, **kw)]


def test_int8_generates_what_the_full_cache_does():
    """Values within a 254th of a block's largest move logits by far less than the greedy choices' distance here."""
    full, small = _greedy(_engine(), PROMPTS, 20), _greedy(_engine(kv_dtype="int8"), PROMPTS, 20)
    same = sum(a == b for x, y in zip(full, small) for a, b in zip(x, y))
    assert all(len(x) == 20 for x in small) and [x[0] for x in full] == [x[0] for x in small] and same >= 40


def test_int8_prefill_attends_to_the_values_that_the_cache_holds():
    """The first token after a prompt and the one after the same prompt and its own continuation agree with a model run
    over the values read back: prefill and decode see one cache."""
    e = _engine(kv_dtype="int8")
    out = _greedy(e, [list(range(40, 75))], 12)[0]
    f = _engine(kv_dtype="int8")
    again = [_greedy(f, [list(range(40, 75)) + out[:i]], 1)[0][0] for i in range(12)]
    assert sum(a == b for a, b in zip(again, out)) >= 11  # appended tokens requantise: a near tie may fall the other way
    assert e.blocks.num_free == e.n_pages - 1


def test_int8_memory():
    full, small = _engine(), _engine(kv_dtype="int8")
    # 16 tokens of a head of 64: 2056 bytes of K, V and scales, against 4096 in two-byte values
    assert small._kv_bytes_per_token() == -(-2 * 2 * (16 * 128 + 8) // 16) and full._kv_bytes_per_token() == 2 * 2 * 256
    assert sum(t.numel() * t.element_size() for c in small.kv for t in c) == 2 * small.n_pages * 2 * (16 * 128 + 8)
    assert all(t.data_ptr() % 16 == 0 for c in small.kv for t in c)
    assert small.mega_reason == "not on CUDA"


@pytest.mark.parametrize("kv_dtype", ["auto", "int8"])
def test_tables_follow_the_pages_of_the_requests(kv_dtype):
    """Rows that grow, finish and move: every running row's table and slot are those of its request's page list."""
    e = _engine(kv_dtype=kv_dtype)
    rids = [e.submit(p, n, temperature=0.0) for p, n in zip(PROMPTS * 2, (3, 40, 25, 9, 60, 5, 33, 17))]
    seen = 0
    while e.has_work():
        e.step()
        for i, req in enumerate(e.running):
            bt = e.st["block_table"][i].tolist()
            assert bt[:len(req.pages)] == req.pages and not any(bt[len(req.pages):])
            pos = int(e.st["pos"][i])
            assert int(e.st["slot"][i]) == req.pages[pos // 16] * 16 + pos % 16
            seen += 1
    assert seen > 20 and all(len(e.finished[r].output_ids) == n for r, n in zip(rids, (3, 40, 25, 9, 60, 5, 33, 17)))
    assert e.blocks.num_free == e.n_pages - 1


@pytest.mark.parametrize("kv_dtype", ["auto", "int8"])
@pytest.mark.parametrize("overrides", [{"rope_scaling": YARN}, {"partial_rotary_factor": 0.5, "rope_interleaved": True}])
def test_scaled_positions_in_engine_and_model_agree(overrides, kv_dtype):
    e = _engine(overrides, kv_dtype=kv_dtype)
    g = e.generate([list(range(40, 75))], 16, temperature=1.0, ignore_eos=True)[0]
    ids = torch.tensor(g.tokens)
    n = len(ids)
    lp = torch.log_softmax(e.model.logits(ids, torch.arange(n, dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32), n), -1)
    want = lp[torch.arange(34, n - 1), ids[35:]]
    got = torch.tensor(g.output_logprobs)
    assert torch.allclose(got, want, atol=1e-4 if kv_dtype == "auto" else 3e-2)
    # and they are not the plain positions'
    plain = build_model(get_model_args("qwen3", "debugmodel"), seed=3)
    other = torch.log_softmax(plain.logits(ids, torch.arange(n, dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32), n), -1)
    assert not torch.allclose(got, other[torch.arange(34, n - 1), ids[35:]], atol=3e-2)


def test_a_row_that_reserves_more_pages_than_its_table_has():
    """A prompt and its tokens that end with the longest sequence reserve a page for one token more."""
    from meshy_b200.ops import checks

    e = _engine(kv_dtype="int8")
    checks.set_enabled(True)
    try:
        g = e.generate([list(range(100, 100 + 250)), [1, 2]], 6, temperature=0.0)
    finally:
        checks.set_enabled(False)
    assert [len(x.output_ids) for x in g] == [6, 6] and e.blocks.num_free == e.n_pages - 1


def test_int8_with_controls_and_interruption():
    e = _engine(kv_dtype="int8")
    out = _greedy(e, PROMPTS, 9, allowed_tokens=[7, 8, 2000], repetition_penalty=1.3)
    assert all(set(o) <= {7, 8, 2000} for o in out)
    rids = [e.submit(p, 50, temperature=0.0) for p in PROMPTS]
    e.step()
    part = {g.rid: g for g in e.abort_all()}
    assert set(part) == set(rids) and e.blocks.num_free == e.n_pages - 1
    assert _greedy(e, PROMPTS, 5) == _greedy(_engine(kv_dtype="int8"), PROMPTS, 5)


def test_refusals_and_command_line():
    from meshy_b200.rollout import server
    from meshy_b200.service.inference import server_args_to_cli

    args = get_model_args("qwen3", "debugmodel")
    with pytest.raises(ValueError, match="kv_dtype"):
        RolloutEngine(args, max_running=2, max_total_tokens=256, kv_dtype="fp8")
    with pytest.raises(ValueError, match="multiple of 16"):
        RolloutEngine(args, max_running=2, max_total_tokens=256, page_size=24, kv_dtype="int8")
    cli = server_args_to_cli({"kv_cache_dtype": "int8", "json_model_override_args": {"rope_scaling": YARN}})
    assert cli[:2] == ["--json-model-override-args", '{"rope_scaling": ' + '{"rope_type": "yarn", "factor": 4.0, '
                       '"original_max_position_embeddings": 64}}'] and cli[2:] == ["--kv-cache-dtype", "int8"]
    assert server._json_object('{"rope_theta": 2}') == {"rope_theta": 2}
    with pytest.raises(Exception, match="JSON object"):
        server._json_object("[1]")
