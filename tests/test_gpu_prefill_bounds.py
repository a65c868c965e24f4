"""max_q_len is an upper bound of a sequence's query rows: a loose one, up to the largest, changes nothing."""
import pytest
import torch

import localstack_b200 as L
from tests.bounded_ref import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_q", [71, 10000, 1 << 30, 2**31 - 1])
@pytest.mark.parametrize("kind", ["plain", "window", "window_q8"])
@pytest.mark.parametrize("seqs", [[(0, 70, 70), (900, 3, 903)], [(30, 70, 100)]])
def test_loose_bounds(seqs, kind, max_q):
    q8 = kind == "window_q8"
    T = sum(t for _, t, _ in seqs)
    b = Batch([n for _, _, n in seqs], 16, 4, seed=T, q8=q8, n_q=T, q_dtype=torch.float32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    start = [0]
    for _, t, _ in seqs:
        start.append(start[-1] + t)
    args = (*b.cache, b.q, i32(start), i32([p for p, _, _ in seqs]), b.lens_t, b.bt)

    def run(bound):
        if kind == "plain":
            return L.attn_prefill(*args, bound)
        return (L.attn_prefill_window_q8 if q8 else L.attn_prefill_window)(*args, bound, 200, 4)

    # the bound decides whether a call is split along the keys: loose ones count as many tiles as the tokens fill
    want, got = run(T), run(max_q)
    L.check_status()
    assert torch.equal(got, want)
    if kind == "window":
        assert (L.prefill_window_workspace_bytes(b.q, 4, max_q, b.bt, 200, 4)
                == L.prefill_window_workspace_bytes(b.q, 4, T, b.bt, 200, 4))
