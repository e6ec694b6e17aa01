"""Logit controls on the CPU: formulas against plain Python, the token state, and refusals."""

import math

import pytest
import torch

from meshy_b200.ops import controls as C


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_bits():
    b = C.token_bits([0, 31, 32, 63, 64], 70)
    assert b.shape == (3,) and (b.to(torch.int64) & 0xFFFFFFFF).tolist() == [0x80000001, 0x80000001, 1]
    with pytest.raises(ValueError):
        C.token_bits([70], 70)


def test_formula():
    V = 70
    ctl = C.LogitControls.create(3, V, device="cpu", max_bias=2)
    ctl.set_slot(1, repetition_penalty=1.5, frequency_penalty=0.25, presence_penalty=0.5, logit_bias={3: 2.0, 69: -1.0},
                 allowed_tokens=[0, 3, 31, 32, 69])
    prompt, output = [0, 5, 69], [3, 3, 31, 0]
    C.load_tokens(ctl, torch.tensor([1]), torch.tensor(prompt + output), _ints(0, 7), _ints(3))
    z = torch.linspace(-3, 3, V)[None].repeat(2, 1)
    raw = z.clone()
    out = C.apply_logit_controls(z, ctl, torch.tensor([1, -1]), new_tokens=torch.tensor([32, 4]))
    assert out.data_ptr() == z.data_ptr() and torch.equal(out[1], raw[1])
    output = output + [32]
    for v in range(V):
        x, n = float(raw[0, v]), output.count(v)
        if v in prompt or n:
            x = x / 1.5 if x > 0 else x * 1.5
        x = x - 0.25 * n - (0.5 if n else 0.0) + {3: 2.0, 69: -1.0}.get(v, 0.0)
        x = x if v in (0, 3, 31, 32, 69) else -math.inf
        assert float(out[0, v]) == pytest.approx(x, abs=1e-5)


def test_out_that_shares_memory_with_the_logits():
    ctl = C.LogitControls.create(2, 8, device="cpu", max_bias=1)
    ctl.set_slot(0, logit_bias={3: 2.0})
    room = torch.arange(24.0)
    z = room[:16].view(2, 8).clone()
    out = C.apply_logit_controls(room[:16].view(2, 8), ctl, torch.tensor([0, 1]), out=room[8:].view(2, 8))
    z[0, 3] += 2.0
    assert torch.equal(out, z)


def test_done_rows_and_unused_slots():
    ctl = C.LogitControls.create(2, 40, device="cpu", max_bias=0)
    C.load_tokens(ctl, torch.tensor([0, -1]), torch.tensor([1, 2, 99, -4]), _ints(0, 4, 4), _ints(1, 0))
    assert ctl.counts[0].nonzero().flatten().tolist() == [2] and int(ctl.seen[0, 0]) == 0b110 and int(ctl.counts[1].sum()) == 0
    z = torch.zeros(2, 40)
    C.apply_logit_controls(z, ctl, torch.tensor([0, 1]), new_tokens=torch.tensor([7, 8]), done=_ints(1, 0))
    assert int(ctl.counts[0, 7]) == 0 and int(ctl.counts[1, 8]) == 1


@pytest.mark.parametrize("kw", [dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=math.inf),
                                dict(frequency_penalty=math.nan), dict(presence_penalty=math.inf), dict(logit_bias={40: 1.0}),
                                dict(logit_bias={-1: 1.0}), dict(logit_bias={1: math.inf}), dict(logit_bias={1: 0., 2: 0., 3: 0.}),
                                dict(logit_bias={1: 0., "1": 0.}), dict(allowed_tokens=[]), dict(allowed_tokens=[40])])
def test_values_are_refused(kw):
    ctl = C.LogitControls.create(1, 40, device="cpu", max_bias=2)
    with pytest.raises(ValueError):
        ctl.set_slot(0, **kw)


@pytest.mark.parametrize("kw", [dict(repetition_penalty=1e39), dict(repetition_penalty=1e-50), dict(repetition_penalty=math.nan),
                                dict(frequency_penalty=1e39), dict(presence_penalty=-1e39), dict(logit_bias={1: -1e39})])
def test_values_outside_fp32_are_refused(kw):
    ctl = C.LogitControls.create(1, 40, device="cpu", max_bias=2)
    with pytest.raises(ValueError):
        ctl.set_slot(0, **kw)


def test_slots_and_masks_are_checked():
    ctl = C.LogitControls.create(2, 70, device="cpu", max_bias=0)
    ok = C.token_bits([5], 70)
    for slot, bits in ((0, ok[:1]), (0, ok[None]), (0, ok.long()), (0, ok.bool()), (-1, ok), (2, ok), (-1, None)):
        with pytest.raises(ValueError):
            ctl.set_mask(slot, bits)
    for slot in (-1, 2):
        with pytest.raises(ValueError):
            ctl.set_slot(slot, presence_penalty=1.0)
    assert ctl.mask_on.tolist() == [0, 0] and ctl.presence.tolist() == [0.0, 0.0] and bool((ctl.mask == -1).all())
    ctl.set_mask(1, ok)
    assert ctl.mask[1].tolist() == ok.tolist() and ctl.mask_on.tolist() == [0, 1]


def test_allowed_tokens_may_be_an_iterator():
    ctl = C.LogitControls.create(1, 40, device="cpu", max_bias=0)
    ctl.set_slot(0, allowed_tokens=iter([3, 33]))
    out = C.apply_logit_controls(torch.zeros(1, 40), ctl, torch.tensor([0]))
    assert out[0].isfinite().nonzero().flatten().tolist() == [3, 33]


def test_sizes_are_refused():
    for slots, vocab, k in ((0, 4, 0), (1, 0, 0), (1, 4, -1)):
        with pytest.raises(ValueError):
            C.LogitControls.create(slots, vocab, device="cpu", max_bias=k)
