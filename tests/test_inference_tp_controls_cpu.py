"""Refused requests, logit controls and the 4-bit cache on a tensor-parallel replica (gloo, 2 ranks)."""

import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

PROMPTS = [[3, 14, 15, 92, 65, 35], [8, 97, 93, 23, 84, 62, 64, 33, 83, 27], [2, 71]]
CONTROLS = dict(repetition_penalty=1.3, frequency_penalty=0.2, presence_penalty=0.3, logit_bias={11: 2.0},
                allowed_tokens=list(range(5, 1500)))
UNUSABLE = [dict(repetition_penalty=-1.0), dict(allowed_tokens=[]), dict(logit_bias={5000: 1.0}), dict(n_generated=99),
            dict(temperature="warm"), dict(frequency_penalty=None), dict(logit_bias={float("inf"): 1.0})]


def _engine(group=None, **kw):
    from meshy_b200.models import get_model_args
    from meshy_b200.rollout.engine import RolloutEngine

    return RolloutEngine(get_model_args("qwen3", "debugmodel"), device="cpu", max_running=8, max_seq_len=128, seed=0,
                         sync_every=4, tp_group=group, **kw)


def _run(eng, **kw):
    gens = eng.generate(PROMPTS, [12, 7, 20], temperature=0.0, ignore_eos=True, **kw)
    return [g.output_ids for g in gens]


def _worker(rank, port, q, what):
    try:
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
        dist.init_process_group("gloo", rank=rank, world_size=2)
        from meshy_b200.rollout.spmd import EngineLeader, follow

        g = dist.group.WORLD
        eng = _engine(g, kv_dtype="int4" if what == "int4" else "auto")
        out = {}
        if rank == 1:
            follow(eng, g)
        else:
            lead = EngineLeader(eng, g)
            if what == "refused":
                out["plain"] = _run(lead)
                for bad in UNUSABLE:
                    for call in (lambda: lead.submit(PROMPTS[0], 4, **bad), lambda: lead.generate(PROMPTS, 4, **bad)):
                        try:
                            call()
                            out["accepted"] = bad
                        except (TypeError, ValueError, OverflowError):
                            pass
                out["again"] = _run(lead)
            else:
                out["controlled"] = _run(lead, **CONTROLS)
                out["plain"] = _run(lead)
            lead.stop()
        # both ranks sampled, so both hold every token
        q.put((rank, dict(out, tokens=eng.st["out_tok"].tolist(), waiting=len(eng.waiting))))
        dist.barrier()
        dist.destroy_process_group()
    except Exception:
        import traceback

        q.put((rank, traceback.format_exc()))


def _two_ranks(what):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ps = [ctx.Process(target=_worker, args=(r, port, q, what)) for r in range(2)]
    for p in ps:
        p.start()
    res = dict(q.get(timeout=240) for _ in range(2))
    for p in ps:
        p.join(timeout=60)
    for v in res.values():
        assert isinstance(v, dict), v
    assert res[0]["tokens"] == res[1]["tokens"] and res[0]["waiting"] == res[1]["waiting"] == 0
    return res[0]


@pytest.mark.timeout(300)
def test_a_refused_request_leaves_the_replica_serving():
    out = _two_ranks("refused")
    assert "accepted" not in out
    assert out["plain"] == out["again"] == _run(_engine())


@pytest.mark.timeout(300)
@pytest.mark.parametrize("what", ["auto", "int4"])
def test_controls_on_a_replica(what):
    out = _two_ranks(what)
    assert all(5 <= t < 1500 for o in out["controlled"] for t in o) and out["controlled"] != out["plain"]
    if what == "auto":  # (4-bit keys and values of sums in another order may land on another nibble)
        assert out["controlled"] == _run(_engine(), **CONTROLS) and out["plain"] == _run(_engine())
