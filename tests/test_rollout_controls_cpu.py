"""Rollout engine with a 4-bit KV cache and with logit controls, on the CPU (fp32 model, exact references)."""

import asyncio

import pytest
import torch

from meshy_b200.models import build_model, get_model_args
from meshy_b200.rollout.engine import RolloutEngine

PROMPTS = [[5, 9, 77, 300, 12], [1, 2, 3], list(range(40, 75))]


def _engine(**kw):
    args = get_model_args("qwen3", "debugmodel")
    model = build_model(args, seed=3)
    return RolloutEngine(args, model=model, max_running=4, max_total_tokens=2048, max_seq_len=256, page_size=16,
                         sync_every=3, **kw)


def _greedy(e, prompts, n, **kw):
    return [g.output_ids for g in e.generate(prompts, n, temperature=0.0, **kw)]


def test_int4_prefill_and_decode_see_the_same_cache():
    """A continuation prefills what the first run decoded: the tokens have to go on as if nothing happened."""
    whole = _greedy(_engine(kv_dtype="int4"), PROMPTS, 24)
    e = _engine(kv_dtype="int4")
    first = _greedy(e, PROMPTS, 11)
    rest = _greedy(e, [p + f for p, f in zip(PROMPTS, first)], 13)
    assert [f + r for f, r in zip(first, rest)] == whole
    assert e.blocks.num_free == e.n_pages - 1


def test_int4_takes_a_fraction_of_the_memory():
    full, small = _engine(), _engine(kv_dtype="int4")
    assert small._kv_bytes_per_token() * 256 == full._kv_bytes_per_token() * 72  # head width 64, against two bytes a value
    assert sum(t.numel() * t.element_size() for c in small.kv for t in c) == small.n_pages * 16 * small._kv_bytes_per_token()


def test_allowed_tokens_and_bias():
    e = _engine()
    out = _greedy(e, PROMPTS, 9, allowed_tokens=[7, 8, 2000])
    assert all(set(o) <= {7, 8, 2000} for o in out)
    out = _greedy(e, PROMPTS, 4, logit_bias={123: 1e4})
    assert out == [[123] * 4] * 3


@pytest.mark.parametrize("kind", ["array", "tensor", "range", "set", "iterator"])
def test_allowed_tokens_of_any_kind(kind):
    np = pytest.importorskip("numpy")
    ids = [7, 8, 9]
    allowed = {"array": np.array(ids), "tensor": torch.tensor(ids), "range": range(7, 10), "set": set(ids), "iterator": iter(ids)}[kind]
    e = _engine()
    rid = e.submit(PROMPTS[0], 6, temperature=0.0, allowed_tokens=allowed)
    e.run_until_idle()
    assert set(e.finished[rid].output_ids) <= set(ids)


def test_controls_changed_after_submit_do_not_reach_the_request():
    e = _engine()
    allowed, bias = [7, 8], {7: 1e4}
    rid = e.submit(PROMPTS[0], 3, temperature=0.0, allowed_tokens=allowed, logit_bias=bias)
    allowed[:] = [10 ** 6]
    bias[-1] = 0.0
    e.run_until_idle()
    assert e.finished[rid].output_ids == [7] * 3


def test_presence_penalty_never_repeats_and_continues():
    e = _engine()
    out = _greedy(e, PROMPTS, 20, presence_penalty=1e4)
    assert all(len(set(o)) == 20 for o in out)
    # a continued request counts its earlier output (and only that: prompts may be repeated)
    more = [_greedy(e, [p + o], 10, presence_penalty=1e4, n_generated=len(o))[0] for p, o in zip(PROMPTS, out)]
    assert all(not set(o) & set(m) for o, m in zip(out, more))
    assert [o + m for o, m in zip(out, more)] == _greedy(_engine(), PROMPTS, 30, presence_penalty=1e4)


def test_logprobs_are_the_controlled_distribution():
    e = _engine()
    g = e.generate([PROMPTS[0]], 3, temperature=0.7, repetition_penalty=1.7, frequency_penalty=0.4, allowed_tokens=range(0, 2048, 2))[0]
    seq, args = list(PROMPTS[0]), e.args
    for tok, lp in zip(g.output_ids, g.output_logprobs):
        t = torch.tensor(seq)
        with torch.no_grad():
            z = e.model.logits(t, torch.arange(len(seq), dtype=torch.int32), torch.tensor([0, len(seq)], dtype=torch.int32),
                               len(seq))[-1].double()
        for v in set(seq):
            z[v] = z[v] / 1.7 if z[v] > 0 else z[v] * 1.7
        for v in seq[len(PROMPTS[0]):]:
            z[v] -= 0.4
        z[1::2] = -torch.inf
        assert tok % 2 == 0 and lp == pytest.approx(float(torch.log_softmax(z / 0.7, -1)[tok]), abs=1e-4)
        seq.append(tok)


def test_requests_without_controls_are_not_touched():
    plain = _greedy(_engine(), PROMPTS, 12)
    e = _engine()
    a = e.submit(PROMPTS[0], 12, temperature=0.0)
    b = e.submit(PROMPTS[1], 12, temperature=0.0, presence_penalty=1e4, logit_bias={3: -5.0})
    c = e.submit(PROMPTS[2], 12, temperature=0.0)
    e.run_until_idle()
    assert e.finished[a].output_ids == plain[0] and e.finished[c].output_ids == plain[2]
    assert len(set(e.finished[b].output_ids)) == 12
    assert _greedy(e, PROMPTS, 12) == plain  # its slot serves plain requests again


def test_controls_with_int4_cache_and_filters():
    e = _engine(kv_dtype="int4")
    gens = e.generate(PROMPTS, 15, temperature=1.0, top_k=4, top_p=0.9, allowed_tokens=range(100), repetition_penalty=1.2)
    assert all(max(g.output_ids) < 100 and len(g.output_ids) == 15 for g in gens)
    assert all(torch.isfinite(torch.tensor(g.output_logprobs)).all() for g in gens)


@pytest.mark.parametrize("kw", [dict(repetition_penalty=0.0), dict(logit_bias={5000: 1.0}), dict(allowed_tokens=[]),
                                dict(logit_bias={i: 1.0 for i in range(301)}), dict(n_generated=6), dict(n_generated=-1)])
def test_unusable_values_are_refused(kw):
    e = _engine()
    with pytest.raises(ValueError):
        e.submit(PROMPTS[0], 4, **kw)
    assert not e.waiting


@pytest.mark.parametrize("kv_dtype", ["auto", "int4"])
def test_requests_of_a_prefill_that_raises_are_not_lost(kv_dtype, monkeypatch):
    e = _engine(kv_dtype=kv_dtype)
    want = _greedy(e, PROMPTS, 6, presence_penalty=0.5)
    real = e._sample_rows

    def fails(h, reqs):
        raise RuntimeError("no logits")

    monkeypatch.setattr(e, "_sample_rows", fails)
    rids = [e.submit(p, 6, temperature=0.0, presence_penalty=0.5) for p in PROMPTS]
    free, slots = e.blocks.num_free, len(e.free_out_slots)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no logits"):
            e.step()
    assert [r.rid for r in e.waiting] == rids and not e.running
    assert e.blocks.num_free == free and len(e.free_out_slots) == slots and int(e.st["done"].min()) == 1
    monkeypatch.setattr(e, "_sample_rows", real)
    e.run_until_idle()  # served after all
    assert [e.finished.pop(r).output_ids for r in rids] == want
    monkeypatch.setattr(e, "_sample_rows", fails)
    rids = [e.submit(p, 6) for p in PROMPTS]
    with pytest.raises(RuntimeError, match="no logits"):
        e.step()
    assert [g.rid for g in e.abort_all()] == rids and not e.has_work()


def test_unknown_kv_dtype_is_refused():
    with pytest.raises(ValueError, match="kv_dtype"):
        _engine(kv_dtype="fp8")


@pytest.mark.parametrize("head_dim,page", [(32, 16), (192, 16), (64, 24)])
def test_unsupported_geometry_of_the_4bit_cache_is_refused(head_dim, page):
    args = get_model_args("qwen3", "debugmodel", head_dim=head_dim)
    model = build_model(args, seed=3)
    with pytest.raises(ValueError, match="4-bit KV cache"):
        RolloutEngine(args, model=model, max_running=4, max_total_tokens=768, max_seq_len=96, page_size=page, kv_dtype="int4")
    RolloutEngine(args, model=model, max_running=4, max_total_tokens=768, max_seq_len=96, page_size=page)


def test_server_takes_the_parameters_and_answers_400():
    pytest.importorskip("aiohttp")
    from aiohttp.test_utils import TestClient, TestServer

    from meshy_b200.rollout.server import EngineRunner, build_app

    async def go():
        runner = EngineRunner(_engine(kv_dtype="int4"))
        async with TestClient(TestServer(build_app(runner))) as c:
            r = await c.post("/generate", json={"input_ids": PROMPTS[0], "return_logprob": True, "sampling_params": {
                "temperature": 0.0, "max_new_tokens": 5, "logit_bias": {"17": 1e4}, "allowed_token_ids": [17, 18],
                "presence_penalty": 0.5, "n_generated": 2}})
            bad = await c.post("/generate", json={"input_ids": PROMPTS[0], "sampling_params": {"repetition_penalty": -1}})
            out = r.status, (await r.json())["output_ids"], bad.status, (await bad.json())["error"]
        runner.shutdown()
        return out

    ok, ids, bad, msg = asyncio.run(go())
    assert ok == 200 and ids == [17] * 5 and bad == 400 and "repetition_penalty" in msg


def test_server_args_key():
    from meshy_b200.service.inference import server_args_to_cli

    assert server_args_to_cli({"kv_cache_dtype": "int4"}) == ["--kv-cache-dtype", "int4"]
