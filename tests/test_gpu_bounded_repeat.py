"""The bounded-cache operators repeat their own bits: the same inputs, over other contents of the workspaces."""
import pytest
import torch

import localstack_b200 as L
from tests.bounded_ref import Batch

pytestmark = pytest.mark.gpu


def _workspaces(n):
    """Fresh bytes of every kind that an earlier call could have left."""
    for fill in (0, 0xff, 0x7f, 0x3c):
        yield torch.full((n,), fill, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("lens", [[513], [5000], [700, 3, 0, 4097], list(range(1, 3000, 61))])
def test_decodes(lens, q8):
    b = Batch(lens, 16, 4, seed=len(lens), q8=q8)
    sfx, width = "_q8" if q8 else "", b.bt.shape[1] * 32
    dec, wts = L.DecodeWorkspace(len(lens), 16, 4), L.WeightsWorkspace(len(lens), 16, 4, width)
    seen = []
    for ws in _workspaces(wts.buf.numel()):
        dec.buf, wts.buf = ws[:dec.buf.numel()], ws
        for _ in range(3):
            acc = torch.zeros(len(lens), width, device="cuda")
            seen.append((*getattr(L, "attn_decode_window" + sfx)(*b.cache, b.q, b.bt, b.lens_t, 300, 4, want_lse=True, workspace=dec),
                         *getattr(L, "attn_decode_weights" + sfx)(*b.cache, b.q, b.bt, b.lens_t, acc, want_lse=True, workspace=wts),
                         acc))
    L.check_status()
    for other in seen[1:]:
        assert all(torch.equal(x, y) for x, y in zip(seen[0], other))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("seqs", [[(0, 900, 900), (3000, 130, 3130)], [(4000, 2, 4002)], [(i, 3, i + 3) for i in range(0, 900, 6)]])
def test_prefill(seqs, q8):
    T = sum(t for _, t, _ in seqs)
    b = Batch([n for _, _, n in seqs], 16, 4, seed=T, q8=q8, n_q=T, q_dtype=torch.float32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    start = [0]
    for _, t, _ in seqs:
        start.append(start[-1] + t)
    longest = max(t for _, t, _ in seqs)
    need = L.prefill_window_workspace_bytes(b.q, 4, longest, b.bt, 1000, 4)
    fn = L.attn_prefill_window_q8 if q8 else L.attn_prefill_window
    args = (*b.cache, b.q, i32(start), i32([p for p, _, _ in seqs]), b.lens_t, b.bt, longest, 1000, 4)
    seen = [fn(*args, workspace=ws) for ws in _workspaces(need) for _ in range(3)]
    L.check_status()
    assert all(torch.equal(seen[0], x) for x in seen[1:])
