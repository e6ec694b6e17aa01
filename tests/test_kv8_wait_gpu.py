"""A wait of the 8-bit attention that gives up: the device error word says so, and the calls that follow on the same workspace
are right without anything being cleared (GPU). The limit of the waits is a number of cycles; with 0 they give up at once."""

import pytest
import torch

from test_kv8_gpu import _filled, _q

pytestmark = pytest.mark.gpu

SHAPES = [(128, 64, 12, 2, [20011]), (128, 64, 12, 2, list(range(1, 8000, 211))), (64, 16, 14, 2, [5001, 0, 17, 3333]),
          (64, 64, 24, 2, [2048] * 40), (128, 32, 8, 8, [700] * 3), (128, 64, 32, 8, [1, 0, 9000] * 20)]


@pytest.fixture
def C():
    from meshy_b200.ops._ext import ext

    assert int(ext().device_error()) == 0
    yield ext()
    ext().clear_device_error()


def _same(a, b):
    """Bit for bit (a row that is longer than its tokens reads scales that are NaN)."""
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


def _case(hd, page, Hq, Hkv, lens):
    c, bt = _filled(lens, Hkv, hd, page)
    return _q(len(lens), Hq, hd), c.k, c.v, c.scale, bt, torch.tensor(lens, dtype=torch.int32, device="cuda"), hd ** -0.5


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}-{len(s[4])}")
def test_calls_after_one_that_gave_up(C, shape):
    args = _case(*shape)
    want = C.kv8_attention(*args)
    for wait in (0, 1, 300, 1000, 3000, 0):  # some CTAs may get through
        C.kv8_attention(*args, wait=wait)
        err = int(C.device_error())
        assert err in ((2, 3) if wait == 0 else (0, 2, 3))
        C.clear_device_error()
        for _ in range(2):
            assert torch.equal(C.kv8_attention(*args), want)
        assert int(C.device_error()) == 0


def test_other_lengths_after_one_that_gave_up(C):
    """Other segments are cut next time: a counter left behind would show."""
    hd, page, Hq, Hkv, lens = SHAPES[1]
    args = list(_case(hd, page, Hq, Hkv, lens))
    lengths = [args[5], args[5].flip(0).contiguous(), args[5] // 3, torch.full_like(args[5], 100)]
    lengths[1] = torch.minimum(lengths[1], args[5])  # (a row's table has pages for its own tokens)
    want = [C.kv8_attention(*args[:5], n, args[6]) for n in lengths]
    for i, n in enumerate(lengths):
        C.kv8_attention(*args[:5], n, args[6], wait=0)
        for m, w in zip(lengths[i:] + lengths[:i], want[i:] + want[:i]):
            assert _same(C.kv8_attention(*args[:5], m, args[6]), w)
    assert int(C.device_error()) in (2, 3)


def test_in_a_captured_graph(C):
    args = _case(*SHAPES[0])
    want = C.kv8_attention(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = C.kv8_attention(*args)
        C.kv8_attention(*args, wait=0)
        second = C.kv8_attention(*args)
    for _ in range(3):
        first.zero_(), second.zero_()
        graph.replay()
        assert int(C.device_error()) in (2, 3)
        C.clear_device_error()
        assert torch.equal(first, want) and torch.equal(second, want)
    assert torch.equal(C.kv8_attention(*args), want) and int(C.device_error()) == 0


def test_beside_calls_on_another_stream(C):
    """Nothing of another stream's workspace is touched."""
    args, others = _case(*SHAPES[0]), _case(*SHAPES[1])
    want = C.kv8_attention(*others)
    torch.cuda.synchronize()
    s, out = torch.cuda.Stream(), []
    for _ in range(50):
        with torch.cuda.stream(s):
            out.append(C.kv8_attention(*others))
        C.kv8_attention(*args, wait=0)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in out) and int(C.device_error()) in (2, 3)
