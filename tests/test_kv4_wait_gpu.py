"""A wait of the 4-bit attention that gives up: the device error word says so, and the calls that follow on the same workspace
are right without anything being cleared (GPU). With a limit of 0 cycles the waits give up at once."""

import pytest
import torch

from test_kv4_gpu import _setup

pytestmark = pytest.mark.gpu

SHAPES = [(128, 64, 12, 2, [20011]), (128, 64, 12, 2, list(range(1, 8000, 211))), (64, 16, 14, 2, [5001, 0, 17, 3333]),
          (64, 64, 24, 2, [2048] * 40), (128, 16, 8, 8, [700] * 3), (64, 32, 32, 8, [1, 0, 9000] * 20)]


@pytest.fixture
def C():
    from meshy_b200.ops._ext import ext

    assert int(ext().device_error()) == 0
    yield ext()
    ext().clear_device_error()


def _case(hd, page, Hq, Hkv, lens):
    q, c, bt, n = _setup(lens, Hq, Hkv, hd, page)
    return q, c.k, c.v, c.scale, bt, n, hd ** -0.5


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}-{len(s[4])}")
def test_calls_after_one_that_gave_up(C, shape):
    args = _case(*shape)
    want = C.kv4_attention(*args)
    shorter = torch.minimum(args[5], args[5].flip(0) // 2 + 1)
    other = C.kv4_attention(*args[:5], shorter, args[6])
    for wait in (0, 1, 300, 1000, 3000, 0):  # some CTAs may get through
        C.kv4_attention(*args, wait=wait)
        err = int(C.device_error())
        assert err in ((2, 3) if wait == 0 else (0, 2, 3))
        C.clear_device_error()
        assert torch.equal(C.kv4_attention(*args[:5], shorter, args[6]), other)
        assert torch.equal(C.kv4_attention(*args), want)
        assert int(C.device_error()) == 0


def test_in_a_captured_graph(C):
    args = _case(*SHAPES[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = C.kv4_attention(*args)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            first = C.kv4_attention(*args)
            C.kv4_attention(*args, wait=0)
            second = C.kv4_attention(*args)
        for _ in range(3):
            first.zero_(), second.zero_()
            graph.replay()
            assert int(C.device_error()) in (2, 3)
            C.clear_device_error()
            assert torch.equal(first, want) and torch.equal(second, want)
    torch.cuda.synchronize()
