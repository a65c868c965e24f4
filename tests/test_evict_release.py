"""KvWeights.release refuses what would leave the row's weights and positions to other tokens (no GPU)."""
import pytest
import torch

import localstack_b200 as L


class _Pages:
    def __init__(self, device="cpu"):
        self.calls, self.device = [], torch.device(device)

    def release(self, slot, keep, stream=None):
        self.calls.append((slot, keep))


def _weights():
    w, pages = L.KvWeights(2, 4, device="cpu"), _Pages()
    w.acc.fill_(1.0)
    w.held[1], w.shift[1] = 50, 9
    return w, pages


@pytest.mark.parametrize("slot,keep", [(1, 1), (1, 49), (2, 0), (-1, 0), (2, 60)])
def test_refusals_change_nothing(slot, keep):
    w, pages = _weights()
    with pytest.raises(ValueError):
        w.release(pages, slot, keep)
    assert not pages.calls and (w.acc == 1).all() and w.held.tolist() == [0, 50] and w.shift.tolist() == [0, 9]


@pytest.mark.parametrize("slot,keep", [(0, 1), (0, 128), (0, 500), (1, 50), (1, 77)])
def test_a_cut_clears_the_weights_behind_it(slot, keep):
    w, pages = _weights()
    w.release(pages, slot, keep)
    assert pages.calls == [(slot, keep)] and (w.acc[slot, :keep] == 1).all() and not w.acc[slot, keep:].any()
    assert (w.acc[1 - slot] == 1).all() and w.held.tolist() == [0, 50] and w.shift.tolist() == [0, 9]


@pytest.mark.parametrize("keep", [0, -3])
def test_a_removal_clears_the_row(keep):
    w, pages = _weights()
    w.release(pages, 1, keep)
    assert pages.calls == [(1, keep)] and not w.acc[1].any() and w.held.tolist() == w.shift.tolist() == [0, 0]
    assert (w.acc[0] == 1).all()
