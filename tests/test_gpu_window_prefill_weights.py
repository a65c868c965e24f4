"""The windowed prefill's softmax weights one by one, to 11 bits (tests/window_prefill_weights.py)."""
import numpy as np
import pytest
import torch

import localstack_b200 as L
from tests.bounded_ref import close, window_mask
from tests.helpers import scattered_block_tables
from tests.window_prefill_weights import SCALE, one_dim_values, quarters, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (16, 2), (4, 4)])
@pytest.mark.parametrize("seqs,window", [([(0, 300, 300), (1000, 70, 1070), (5, 1, 6)], 2), ([(0, 300, 300), (500, 129, 629)], 17),
                                         ([(0, 700, 700), (1900, 260, 2100)], 128), ([(4000, 3, 4003)], 100), ([(999, 1, 1000), (20, 2, 700)], 1000)])
@pytest.mark.parametrize("scale", [SCALE, 0.25])
def test_single_weights(seqs, window, scale, Hq, Hkv):
    rng = np.random.default_rng(window + Hq)
    lens = [n for _, _, n in seqs]
    bt, n_pages = scattered_block_tables(rng, lens)
    ks = [quarters(rng, (n, Hkv, 128)) for n in lens]
    vs = [one_dim_values(rng, n, Hkv) for n in lens]
    k, v = (torch.zeros(n_pages * 32, Hkv, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    for b, n in enumerate(lens):
        p = np.arange(n)
        cells = torch.from_numpy(bt[b, p // 32].astype(np.int64) * 32 + p % 32).cuda()
        k[cells], v[cells] = torch.from_numpy(ks[b]).cuda().half(), torch.from_numpy(vs[b]).cuda().half()
    starts = np.concatenate([[0], np.cumsum([t for _, t, _ in seqs])])
    q = quarters(rng, (int(starts[-1]), Hq, 128))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    args = (k, v, torch.from_numpy(q).cuda().half(), i32(starts.tolist()), i32([p0 for p0, _, _ in seqs]), i32(lens),
            torch.from_numpy(bt).cuda(), max(t for _, t, _ in seqs), window)
    # with a workspace that lets few queries be split along the keys (the last case: up to 8 keys to a dim), and without
    for ws in (None, torch.empty(256, dtype=torch.uint8, device="cuda")):
        for dtype in (torch.float32, torch.bfloat16):
            out = L.attn_prefill_window(*args, scale=float(scale), out_dtype=dtype, workspace=ws).float().cpu().numpy()
            L.check_status()
            for b, (p0, t, n) in enumerate(seqs):
                rows = slice(starts[b], starts[b + 1])
                seen = window_mask(p0 + np.arange(t), n, window, 0)
                want, tol = reference(q[rows], ks[b], vs[b], seen, scale)
                close(out[rows], want, tol, dtype == torch.bfloat16, f"sequence {b}")
