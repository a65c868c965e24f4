"""Cutting a prompt: its last queries, given to attn_decode_weights as rows over the same pages, weigh its keys
for the eviction; without them every weight is zero."""
import numpy as np
import pytest
import torch

import localstack_b200 as L
from tests.bounded_ref import Batch, attend, close, window_mask
from tests.test_gpu_evict import select_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("n,R", [(700, 16), (97, 1), (2049, 40)])
def test_a_prompts_last_queries_weigh_its_keys(n, R, q8):
    Hq, Hkv = 16, 4
    b = Batch([n], Hq, Hkv, seed=n, q8=q8, n_q=R)  # the queries at positions n - R .. n - 1
    cells = b.bt.shape[1] * 32
    at = torch.arange(n - R, n, dtype=torch.int32, device="cuda")
    w = L.KvWeights(1, b.bt.shape[1])
    rows = torch.zeros(R, cells, device="cuda")
    fn = L.attn_decode_weights_q8 if q8 else L.attn_decode_weights
    out = fn(*b.cache, b.q, b.bt.expand(R, -1).contiguous(), at + 1, rows)
    w.acc[0, :cells] += rows.sum(0)
    L.check_status()
    c = b.cells(0)
    o, _, want, t_o, _, t_w = attend(b.q_host, b.k_host[c], b.v_host[c], window_mask(at.cpu().numpy(), n, 1 << 30, 0), q8)
    close(out.cpu().numpy(), o, t_o)
    acc = w.acc.cpu().numpy()
    # each row's sum over Hq heads, and the sum over R rows, in f32
    close(acc[0, :n], want, t_w + (Hq + R + 1) * 2.0 ** -24 * want, what="weights")
    assert not acc[0, n:].any()
    budget, n_sink, n_recent = n // 3, 2, n // 8
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    m = w.select(lens, budget, n_sink, n_recent)
    s, d = select_ref(acc, np.zeros_like(acc, np.int32), [0], [0], [n], budget, n_sink, n_recent)[0]
    assert m.src[0, :m.n[0]].tolist() == s and m.dst[0, :m.n[0]].tolist() == d
    kept = np.setdiff1d(np.arange(budget), d).tolist() + s
    lost = np.setdiff1d(np.arange(n), kept)
    free = [i for i in kept if n_sink <= i < n - n_recent]
    # no dropped key outweighs a kept one that was not protected (by more than both bounds)
    assert want[lost].max() <= want[free].min() + 2 * t_w.max() + 2.0 ** -18 * want.max()
    # without the queries: the protected keys and the lowest indexes
    w.acc.zero_()
    m = w.select(lens, budget, n_sink, n_recent)
    assert np.setdiff1d(np.arange(budget), m.dst[0, :m.n[0]].tolist()).tolist() == list(range(budget - n_recent))
