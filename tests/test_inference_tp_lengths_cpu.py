"""Prompts that do not fit, on a tensor-parallel replica: both ranks refuse them and go on together (gloo, 2 ranks)."""

import os
import socket

import torch.distributed as dist
import torch.multiprocessing as mp

from test_inference_tp_controls_cpu import PROMPTS, _engine, _run

FULL = [(5 * i) % 900 + 3 for i in range(128)]  # as long as the longest sequence


def _worker(rank, port, q):
    try:
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
        dist.init_process_group("gloo", rank=rank, world_size=2)
        from meshy_b200.rollout.spmd import EngineLeader, follow

        g = dist.group.WORLD
        eng = _engine(g, kv_dtype="int8")
        out = {}
        if rank == 1:
            follow(eng, g)
        else:
            lead = EngineLeader(eng, g)
            out["plain"] = _run(lead)
            out["refused"] = 0
            for call in (lambda: lead.submit(FULL + [1], 4), lambda: lead.generate(PROMPTS + [FULL + [1]], 4),
                         lambda: lead.generate([[1] * 500], 4)):
                try:
                    call()
                except ValueError:
                    out["refused"] += 1
            out["again"] = _run(lead)
            out["full"] = [len(x.output_ids) for x in lead.generate([FULL, PROMPTS[0]], 6, temperature=0.0, ignore_eos=True)]
            lead.stop()
        q.put((rank, dict(out, tokens=eng.st["out_tok"].tolist(), waiting=len(eng.waiting), free=eng.blocks.num_free,
                          pages=eng.n_pages)))
        dist.barrier()
        dist.destroy_process_group()
    except Exception:
        import traceback

        q.put((rank, traceback.format_exc()))


def test_both_ranks_refuse_together():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ps = [ctx.Process(target=_worker, args=(r, port, q)) for r in range(2)]
    for p in ps:
        p.start()
    res = dict(q.get(timeout=240) for _ in range(2))
    for p in ps:
        p.join(timeout=60)
    for v in res.values():
        assert isinstance(v, dict), v
    lead, other = res[0], res[1]
    assert lead["refused"] == 3 and lead["again"] == lead["plain"] and lead["full"] == [1, 6]
    assert lead["tokens"] == other["tokens"]
    assert all(r["waiting"] == 0 and r["free"] == r["pages"] - 1 for r in (lead, other))
