"""KvWeights refuses pages of another device before any call: the kernels would read host memory (no GPU)."""
import pytest
import torch

import localstack_b200 as L


class _Pages:
    device = torch.device("cuda", 0)

    @property
    def state(self):
        raise AssertionError("the library must not be called")

    def release(self, *a, **k):
        raise AssertionError("the library must not be called")


def test_pages_and_weights_on_two_devices():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    w = L.KvWeights(2, 4, device="cpu")
    with pytest.raises(ValueError):
        w.finish(_Pages(), L.KvMoves(i32(2), i32(2, 64), i32(2, 64), 64))
    w.acc.fill_(1.0)
    for keep in (0, 10):
        with pytest.raises(ValueError):
            w.release(_Pages(), 0, keep)
    assert (w.acc == 1).all()
