"""Prompts around the longest sequence of a rollout engine, on the CPU: what does not fit the block table is refused, and
no write gets a slot outside the cache, no attention a length past the table."""

import asyncio

import pytest
import torch

from meshy_b200.models import build_model, get_model_args
from meshy_b200.ops import checks
from meshy_b200.rollout import engine as E

PAGE = 16


@pytest.fixture
def checked():
    """Every index in front of the kernels is checked: slots, tables and lengths outside raise."""
    checks.set_enabled(True)
    yield
    checks.set_enabled(False)


def _engine(kv_dtype="auto", max_seq_len=64, **kw):
    args = get_model_args("qwen3", "debugmodel")
    return E.RolloutEngine(args, model=build_model(args, seed=3), max_running=4, max_total_tokens=1024,
                           max_seq_len=max_seq_len, page_size=PAGE, sync_every=3, kv_dtype=kv_dtype, **kw)


def _watch(monkeypatch):
    """The slots that prefill and decode hand to the cache writes."""
    seen = []

    def spy(at, name, index):
        plain = getattr(at, name)

        def call(*a, **k):
            seen.append(a[index].clone())
            return plain(*a, **k)

        monkeypatch.setattr(at, name, staticmethod(call) if isinstance(at, type) else call)

    spy(E.D, "qkv_rope_to_cache", 11)
    spy(E._KV4, "write", 3)
    spy(E._KV8, "write", 3)
    return seen


@pytest.mark.parametrize("kv_dtype", ["auto", "int4", "int8"])
@pytest.mark.parametrize("n", [62, 63, 64])
def test_prompts_up_to_the_longest_sequence(monkeypatch, checked, kv_dtype, n):
    """They get the tokens that fit, one at least; beside them a row that goes on is not disturbed."""
    prompt = [(7 * i) % 900 + 3 for i in range(n)]
    seen = _watch(monkeypatch)
    e = _engine(kv_dtype)
    long, short = e.generate([prompt, [1, 2, 3]], 9, temperature=0.0)
    assert len(long.output_ids) == max(1, 64 - n) and len(short.output_ids) == 9
    assert seen and min(int(s.min()) for s in seen) >= 0
    assert max(int(s.max()) for s in seen) < e.n_pages * PAGE and e.blocks.num_free == e.n_pages - 1
    assert int(e.st["seq_lens"].max()) <= 64
    # the first token is that of an engine with room to spare, and so is the short row's text
    wide = _engine(kv_dtype, max_seq_len=256)
    first, rest = wide.generate([prompt, [1, 2, 3]], [1, 9], temperature=0.0)
    assert first.output_ids[0] == long.output_ids[0] and rest.output_ids == short.output_ids
    assert torch.allclose(torch.tensor(first.output_logprobs[0]), torch.tensor(long.output_logprobs[0]), atol=1e-5)


@pytest.mark.parametrize("kv_dtype", ["auto", "int4", "int8"])
@pytest.mark.parametrize("n", [65, 66, 200])
def test_longer_prompts_are_refused(kv_dtype, n):
    e = _engine(kv_dtype)
    with pytest.raises(ValueError, match=f"a prompt of {n} tokens is longer than the 64"):
        e.submit([1] * n, 4)
    with pytest.raises(ValueError, match="longer than the 64"):
        e.generate([[1, 2], [1] * n], 4)
    with pytest.raises(ValueError, match="longer than the 64"):
        e.generate([[1, 2], [3], [1] * n, [4]], [4, 4, 4, 4])
    assert not e.waiting and not e.has_work()  # the prompts before it are not left in the queue
    e.submit([9], 2, rid="other")
    with pytest.raises(ValueError, match="longer than the 64"):
        e.generate([[1, 2], [1] * n], 4)
    assert [r.rid for r in e.waiting] == ["other"]
    e.abort_all()
    e.finished.clear()
    assert e.blocks.num_free == e.n_pages - 1
    assert len(e.generate([[1, 2]], 4, temperature=0.0)[0].output_ids) == 4


def test_a_last_page_that_is_begun_holds_prompts(checked):
    """The table has whole pages: a prompt longer than ``max_seq_len`` that they hold gets one token."""
    e = _engine("int8", max_seq_len=50)
    for n in (49, 50, 51, 64):
        assert len(e.generate([[5] * n], 9, temperature=0.0)[0].output_ids) == 1
    with pytest.raises(ValueError, match="longer than the 64"):
        e.submit([5] * 65, 9)


def test_the_server_answers_400():
    from aiohttp.test_utils import TestClient, TestServer

    from meshy_b200.rollout.server import EngineRunner, build_app

    runner = EngineRunner(_engine("int8"))

    async def ask():
        async with TestClient(TestServer(build_app(runner))) as c:
            out = []
            for n in (65, 64):
                r = await c.post("/generate", json={"input_ids": [4] * n, "sampling_params": {"max_new_tokens": 5}})
                out.append((r.status, await r.json()))
            return out

    try:
        (bad, why), (good, answer) = asyncio.run(ask())
    finally:
        runner.shutdown()
    assert bad == 400 and "longer than the 64" in why["error"]
    assert good == 200 and len(answer["output_ids"]) == 1
