"""EngineClient against a server whose engine refuses requests or aborts them half way."""

import asyncio

import pytest

from meshy_b200.engine.rollout_client import EngineClient, _Base

PROMPT = [5, 9, 77, 300, 12]


def _with_server(use, **client):
    """Result of ``use(client, counts)`` against a server over a small CPU engine; ``counts["posts"]``: requests it has seen."""
    pytest.importorskip("aiohttp")
    from aiohttp.test_utils import TestServer

    from meshy_b200.models import build_model, get_model_args
    from meshy_b200.rollout.engine import RolloutEngine
    from meshy_b200.rollout.server import EngineRunner, build_app

    async def go():
        args = get_model_args("qwen3", "debugmodel")
        e = RolloutEngine(args, model=build_model(args, seed=3), max_running=4, max_total_tokens=2048, max_seq_len=256, page_size=16)
        runner = EngineRunner(e)
        app = build_app(runner)
        counts = {"posts": 0}

        async def count(req, resp):
            counts["posts"] += req.path == "/generate"

        app.on_response_prepare.append(count)
        async with TestServer(app) as s:
            c = EngineClient(str(s.make_url("/")).rstrip("/"), attempts=4, backoff=0.2, **client)
            try:
                return await use(c, counts)
            finally:
                await c.close()
                runner.shutdown()

    return asyncio.run(go())


@pytest.mark.parametrize("params", [dict(repetition_penalty=-1), dict(logit_bias={"99999": 1.0}), dict(allowed_token_ids=[])])
def test_a_refused_request_is_not_sent_again(params):
    async def use(c, counts):
        with pytest.raises(ValueError, match="refused.*" + {"allowed_token_ids": "allowed_tokens"}.get(*[next(iter(params))] * 2)):
            await c.generate(PROMPT, dict(params, max_new_tokens=4))
        ok = await c.generate(PROMPT, dict(max_new_tokens=4, temperature=0.0, ignore_eos=True))
        return counts["posts"], ok.output_ids

    posts, ids = _with_server(use)
    assert posts == 2 and len(ids) == 4


@pytest.mark.parametrize("params", [dict(logit_bias=[3, 4]), dict(allowed_token_ids=5), dict(presence_penalty=[1]),
                                    dict(allowed_token_ids=[None]), dict(logit_bias={"a": 1}),
                                    dict(allowed_token_ids=[float("inf")])])
def test_parameters_of_another_type_are_refused(params):
    async def use(c, counts):
        with pytest.raises(ValueError, match="refused"):
            await c.generate(PROMPT, dict(params, max_new_tokens=4))
        return counts["posts"]

    assert _with_server(use) == 1


class _Aborting(_Base):
    """Answers with the given pieces of output, all but the last of them cut off by an abort."""

    def __init__(self, *pieces):
        self.pieces, self.seen = list(pieces), []

    async def _generate_once(self, prompt, params):
        self.seen.append((prompt, params))
        out = self.pieces.pop(0)
        return out, [0.0] * len(out), "abort" if self.pieces else "stop", 0


@pytest.mark.parametrize("before,want", [({}, [None, 2, 3]), ({"n_generated": 4}, [4, 6, 7])])
def test_a_continued_request_keeps_what_was_generated_before(before, want):
    c = _Aborting([1, 2], [3], [4, 5])
    params = dict(before, presence_penalty=0.5, max_new_tokens=9)
    res = asyncio.run(c.generate(PROMPT, params))
    assert res.output_ids == [1, 2, 3, 4, 5] and [p.get("n_generated") for _, p in c.seen] == want
    assert [p for p, _ in c.seen] == [PROMPT, PROMPT + [1, 2], PROMPT + [1, 2, 3]]
    assert params == dict(before, presence_penalty=0.5, max_new_tokens=9)
