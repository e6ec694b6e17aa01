"""What the rollout engine does when a decode kernel reports that one of its waits gave up, with a stub for the device (CPU)."""

import pytest

from meshy_b200.models import build_model, get_model_args
from meshy_b200.ops import _ext
from meshy_b200.rollout.engine import RolloutEngine


class _Device:
    """Stands for the extension: an error word, and the calls made of it."""

    def __init__(self, err):
        self.err, self.calls = err, []

    def __getattr__(self, name):
        def call():
            self.calls.append(name)
            out, self.err = self.err, 0 if name == "clear_device_error" else self.err
            return out

        return call


@pytest.mark.parametrize("kv_dtype", ["int4", "int8"])
def test_an_error_reaches_the_caller_and_the_engine_goes_on(monkeypatch, kv_dtype):
    args = get_model_args("qwen3", "debugmodel")
    e = RolloutEngine(args, model=build_model(args, seed=3), max_running=4, max_total_tokens=1024, max_seq_len=128,
                      page_size=16, sync_every=3, kv_dtype=kv_dtype)
    rids = [e.submit([5, 6, 7], 12, temperature=0.0), e.submit([9] * 20, 12, temperature=0.0)]
    e.step()
    dev = _Device(3)
    with monkeypatch.context() as m:
        m.setattr(_ext, "ext", lambda: dev)
        m.setattr(e, "cuda", True)
        with pytest.raises(RuntimeError, match="device error 3"):
            e._sync_finished()
        # reported once; an engine beside this one keeps its workspaces
        assert dev.calls == ["device_error", "clear_device_error"]
        e._sync_finished()
    assert len(e.running) == 2
    assert {g.rid for g in e.abort_all()} == set(rids) and e.blocks.num_free == e.n_pages - 1
    assert len(e.generate([[5, 6, 7]], 4, temperature=0.0)[0].output_ids) == 4
