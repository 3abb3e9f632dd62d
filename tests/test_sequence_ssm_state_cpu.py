"""CPU-only: a state that does not fit is refused in front of the first layer, so that no layer's state has moved when a step raises."""
import pytest
import torch

import wav2sleep_amd as W


def wrong_states(m, batch):
    """the last layer's is wrong, the first one's right"""
    for change in (lambda c, h: (c[:1], h), lambda c, h: (c, h[:1]), lambda c, h: (c, h[:, :, :8]), lambda c, h: (c.double(), h), lambda c, h: (c, h.half()), lambda c, h: (c,)):
        yield m.init_state(batch)[:-1] + [change(*m.init_state(batch)[-1])]


def test_a_state_that_does_not_fit():
    m = W.SequenceSSM(64, num_layers=2)
    for st in wrong_states(m, 2):
        with pytest.raises(ValueError, match='layer 1'):
            m.step(torch.zeros(2, 64), st)
        with pytest.raises(ValueError, match='layer 1'):
            m.prompt(torch.zeros(2, 3, 64), state=st)


def test_a_step_wants_a_state_that_it_can_write():
    m = W.SequenceSSM(64, num_layers=2)
    for change in (lambda h: h.transpose(1, 2).contiguous().transpose(1, 2), lambda h: h.requires_grad_(True), lambda h: h.to('meta')):
        st = m.init_state(2)
        st[1] = (st[1][0], change(st[1][1]))
        with pytest.raises(ValueError, match='layer 1'):
            m.step(torch.zeros(2, 64), st)
