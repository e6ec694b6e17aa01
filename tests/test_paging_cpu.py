"""Block tables and slot maps from request lengths, on the CPU, against token-by-token counting."""

import random

import pytest
import torch

from meshy_b200.ops import checks
from meshy_b200.ops.paging import TokenMaps, assign_pages, token_maps


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("seed", range(5))
def test_tables_and_maps_token_by_token(seed):
    rng = random.Random(seed)
    page, n, R = rng.choice([1, 7, 16]), rng.randint(1, 9), 12
    start = [rng.randint(0, 40) for _ in range(n)]
    lens = [rng.randint(0, 50) for _ in range(n)]
    rows = rng.sample(range(R), n)
    have, need = [-(-s // page) for s in start], [-(-(s + k) // page) for s, k in zip(start, lens)]
    width = max(need + [1])
    table = torch.randint(1, 1000, (R, width), dtype=torch.int32)
    want = table.tolist()
    free = iter(range(5000, 9000))
    for r, h, m in zip(rows, have, need):
        for j in range(h, m):
            want[r][j] = next(free)
    pages = _i32(range(5000, 5000 + sum(need) - sum(have)))
    assign_pages(table, _i32(rows), _i32(have), _i32(need), pages)
    assert table.tolist() == want
    pos, slots, cu = [], [], [0]
    for r, s, k in zip(rows, start, lens):
        for p in range(s, s + k):
            pos.append(p)
            slots.append(want[r][p // page] * page + p % page)
        cu.append(len(pos))
    out = token_maps(table, _i32(rows), _i32(start), _i32(lens), len(pos) + 2, page)
    assert isinstance(out, TokenMaps)
    assert out.positions.tolist() == pos + [0, 0] and out.slots.tolist() == slots + [-1, -1]
    assert out.cu_seqlens.tolist() == cu and out.slots.dtype == torch.int64
    short = token_maps(table, _i32(rows), _i32(start), _i32(lens), len(pos) // 2, page)
    assert short.slots.tolist() == slots[:len(pos) // 2] and short.cu_seqlens.tolist() == cu


def test_what_falls_outside():
    t = torch.full((2, 3), 7, dtype=torch.int32)
    assign_pages(t, _i32([9, -1, 1]), _i32([0, 0, 2]), _i32([1, 2, 5]), _i32([1, 2, 3, 4, 5, 6, 8, 9]))
    assert t.tolist() == [[7, 7, 7], [7, 7, 4]]  # pages 1, 2, 3 went to rows that there are not, 5 and 6 past the columns
    t[0, 1] = -4
    m = token_maps(t, _i32([0, 5, 0]), _i32([3, 0, -2]), _i32([4, 2, 3]), 9, 4)
    assert m.slots.tolist() == [31, -1, -1, -1, -1, -1, -1, -1, 28]
    assert m.positions.tolist() == [3, 4, 5, 6, 0, 1, -2, -1, 0] and m.cu_seqlens.tolist() == [0, 4, 6, 9]


def test_refusals():
    t, r = torch.zeros(4, 4, dtype=torch.int32), _i32([0, 1])
    for args in ((t.long(), r, r, r, r), (t, r.long(), r, r, r), (t, r, r[:1], r, r), (t, r, r, r, r.long()), (t[0], r, r, r, r),
                 (t, r, r, r, r[None])):
        with pytest.raises(ValueError):
            assign_pages(*args)
    for args in ((t, r, r, r, -1, 16), (t, r, r, r, 4, 0), (t, r, r[:1], r, 4, 16), (t.float(), r, r, r, 4, 16)):
        with pytest.raises(ValueError):
            token_maps(*args)


def test_debug_mode_names_the_row():
    t, r = torch.zeros(4, 4, dtype=torch.int32), _i32([0, 4])
    checks.set_enabled(True)
    try:
        with pytest.raises(IndexError, match="rows"):
            assign_pages(t, r, r, r, r)
        with pytest.raises(IndexError, match="rows"):
            token_maps(t, r, r, r, 4, 16)
        with pytest.raises(IndexError, match="columns"):
            assign_pages(t, _i32([0, 1]), _i32([0, 0]), _i32([5, 1]), _i32([1]))
    finally:
        checks.set_enabled(False)
