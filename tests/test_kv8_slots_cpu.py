"""Debug mode of the 8-bit cache write: what the kernel, whose warps own a block's rows each, leaves undefined is named (CPU)."""

import pytest
import torch

from meshy_b200.ops import checks
from meshy_b200.ops import kv8 as K


@pytest.fixture
def on():
    checks.set_enabled(True)
    yield
    checks.set_enabled(False)


def _write(slots):
    c = K.kv8_empty(5, 1, 16, 64, "cpu")
    x = torch.randn(len(slots), 1, 64).bfloat16()
    K.kv8_write(x, x, c, torch.tensor(slots))
    return c


@pytest.mark.parametrize("slots", [[16, -1, 17], [16, -1, -1, 17], [16, 3, 17], [20, 32, 16], [-1, 40, 41, 30, -1, 42]])
def test_rows_of_a_block_with_others_between_them(on, slots):
    with pytest.raises(IndexError, match="stand together"):
        _write(slots)


@pytest.mark.parametrize("slots", [[16, 16], [40, 41, 40], [-1, 33, 33, -1], [17] * 30])
def test_slots_that_are_given_twice(on, slots):
    with pytest.raises(IndexError, match="given twice"):
        _write(slots)


@pytest.mark.parametrize("slots", [[], [-1], [0, 0, 0], [0, 16, 0, 17 + 16, 0], [17, 16, -1, 40, -1], [5, -1, 5, 64, 79],
                                   [-1, -1, 31, 30, 48, -1]])
def test_what_is_allowed(on, slots):
    _write(slots)


def test_off_by_default():
    _write([16, -1, 17, 16])
