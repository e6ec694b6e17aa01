"""Block tables and slot maps made on the device, against the row-by-row definition."""

import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _compare(table, rows, have, need, pages, start, lens, total, page):
    from meshy_b200.ops import paging, reference as ref

    want = table.clone()
    args = [_i32(x) for x in (rows, have, need, pages)]
    ref.assign_pages(want, *args)
    got = table.cuda()
    paging.assign_pages(got, *(x.cuda() for x in args))
    assert torch.equal(got.cpu(), want)
    maps = [_i32(x) for x in (rows, start, lens)]
    out = paging.token_maps(got, *(x.cuda() for x in maps), total, page)
    for a, b, name in zip(out, ref.token_maps(want, *maps, total, page), out._fields):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b), name


@pytest.mark.parametrize("n, longest, page", [(1, 1, 16), (1, 5000, 64), (7, 300, 16), (255, 40, 48), (256, 90, 1),
                                              (1024, 20, 16), (1025, 13, 64), (5000, 9, 16), (33, 4000, 7)])
@pytest.mark.parametrize("start", [0, 77])
def test_tables_and_maps(n, longest, page, start):
    rng = random.Random(n * 1000 + start)
    lens = [rng.choice([0, 1, longest, rng.randint(0, longest)]) for _ in range(n)]
    R = n + 3
    first = [rng.randint(0, start) for _ in range(n)]
    have = [-(-s // page) for s in first]
    need = [-(-(s + k) // page) for s, k in zip(first, lens)]
    width = max(need + [1])
    table = torch.randint(1, 1 << 20, (R, width), dtype=torch.int32)
    rows = rng.sample(range(R), n)
    pages = [rng.randrange(1 << 30) for _ in range(sum(need) - sum(have))]
    for total in {sum(lens), sum(lens) + 5, max(0, sum(lens) - 3)}:
        _compare(table, rows, have, need, pages, first, lens, total, page)


def test_what_falls_outside():
    table = torch.arange(1, 13, dtype=torch.int32).view(3, 4)
    table[1, 2] = -7
    # rows outside, more pages than columns, fewer pages than wanted, counts below zero
    _compare(table, [5, -1, 0, 1, 2], [0, 0, 3, 2, -2], [2, 1, 9, 1, 3], list(range(100, 110)), [0, 0, 60, 40, -2],
             [5, 5, 10, -4, 6], 40, 16)
    # a page id below zero, a position at the end of int32, a start past the table
    _compare(table, [1, 0, 2], [0, 0, 0], [0, 0, 0], [], [30, (1 << 31) - 3, 64], [20, 6, 3], 40, 16)
    _compare(table, [], [], [], [], [], [], 3, 16)
    _compare(table, [0], [0], [0], [], [0], [0], 0, 16)
    _compare(table[:, :0], [0, 1], [0, 0], [1, 2], [5, 6, 7], [0, 3], [4, 2], 6, 16)
    # a table that is part of a larger one
    wide = torch.arange(60, dtype=torch.int32).view(3, 20)
    _compare(wide[:, 3:9], [2, 0], [1, 0], [3, 2], [901, 902, 903, 904], [10, 0], [30, 20], 50, 16)


def test_sums_past_int32():
    """Offsets saturate; what fits the result is right."""
    from meshy_b200.ops import paging, reference as ref

    big = (1 << 31) - 1
    table = torch.randint(1, 99, (3, 4), dtype=torch.int32)
    args = [_i32(x) for x in ([0, 1, 2], [3, 0, 0], [5, big, big])]
    out = paging.token_maps(table.cuda(), *(x.cuda() for x in args), 40, 16)
    assert out.cu_seqlens.tolist() == [0, 5, big, big]
    want = ref.token_maps(table, _i32([0, 1]), _i32([3, 0]), _i32([5, 35]), 40, 16)
    assert torch.equal(out.slots.cpu(), want[1]) and torch.equal(out.positions.cpu(), want[0])


def test_capture_follows_lengths():
    from meshy_b200.ops import paging, reference as ref

    table = torch.zeros(8, 6, dtype=torch.int32, device="cuda")
    rows, have, need, lens = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in
                              ([3, 1, 6], [0, 0, 0], [2, 1, 3], [20, 16, 40]))
    start = torch.zeros_like(lens)
    pages = torch.arange(1, 20, dtype=torch.int32, device="cuda")

    def step():
        paging.assign_pages(table, rows, have, need, pages)
        return paging.token_maps(table, rows, start, lens, 100, 16)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for new in ([2, 1, 3], [1, 3, 1], [0, 0, 6]):
        need.copy_(torch.tensor(new, dtype=torch.int32))
        lens.copy_(need * 16 - (need > 0).int())
        table.zero_()
        graph.replay()
        want = torch.zeros(8, 6, dtype=torch.int32)
        ref.assign_pages(want, *(x.cpu() for x in (rows, have, need, pages)))
        assert torch.equal(table.cpu(), want)
        for a, b in zip(out, ref.token_maps(want, *(x.cpu() for x in (rows, start, lens)), 100, 16)):
            assert torch.equal(a.cpu(), b)


def test_refusals():
    from meshy_b200.ops import paging

    t = torch.zeros(4, 4, dtype=torch.int32, device="cuda")
    r = torch.arange(2, dtype=torch.int32, device="cuda")
    for args in ((t.long(), r, r, r, r), (t, r.long(), r, r, r), (t, r, r[:1], r, r), (t, r, r, r, r.long()),
                 (t[0], r, r, r, r), (t, r, r, r, r[None])):
        with pytest.raises(ValueError):
            paging.assign_pages(*args)
    for args in ((t, r, r, r, -1, 16), (t, r, r, r, 4, 0), (t, r, r[:1], r, 4, 16), (t.float(), r, r, r, 4, 16)):
        with pytest.raises(ValueError):
            paging.token_maps(*args)
    for args in ((t.t().contiguous().t(), r, r, r, r), (t, r.cpu(), r, r, r), (t, r, r, r, r.cpu())):
        with pytest.raises(RuntimeError):
            paging.assign_pages(*args)
    with pytest.raises(RuntimeError):
        paging.token_maps(t, r, r, r, 1 << 31, 16)
