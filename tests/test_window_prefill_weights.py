"""The bound on single softmax weights (tests/window_prefill_weights.py), on CPU: the kernel's arithmetic lies within
it, and scores that lose bits do not."""
import numpy as np
import pytest

from tests.bounded_ref import window_mask
from tests.window_prefill_weights import SCALE, one_dim_values, quarters, reference, restated


@pytest.mark.parametrize("window", [2, 17, 128])
@pytest.mark.parametrize("scale", [SCALE, 0.25])
def test_the_bound_tells_f32_scores_from_f16_scores(window, scale):
    rng = np.random.default_rng(window)
    q, k, v = quarters(rng, (200, 4, 128)), quarters(rng, (200, 2, 128)), one_dim_values(rng, 200, 2)
    seen = window_mask(np.arange(200), 200, window, 0)
    want, tol = reference(q, k, v, seen, scale)
    ratio = lambda f16: (np.abs(restated(q, k, v, seen, scale, f16) - want) / (tol + 1e-30)).max()  # noqa: E731
    assert ratio(False) <= 1.0
    assert ratio(True) > 1.5
