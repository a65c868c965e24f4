"""The q8_0 query of the bounded-cache decodes: its block scale is amax * (1 / 127) in f32, attn_decode_q8's is
amax / 127. Where the two give the same integers and f16 scales, the same bits come out."""
import numpy as np
import pytest
import torch

import localstack_b200 as L
from tests.bounded_ref import Batch, quantise_q8

pytestmark = pytest.mark.gpu

LENS = [0, 1, 31, 32, 33, 64, 100, 257, 1000, 3000]


def _same(q):
    """Per row [B][Hq] of f32 values: both scales quantise it alike."""
    (a, da), (b, db) = quantise_q8(q, product=True), quantise_q8(q)
    return ((a == b).all(-1) & (da == db).all(-1))


@pytest.mark.parametrize("q_dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv", [(32, 4), (16, 8), (12, 2)])
def test_a_window_over_everything_and_weights_are_attn_decode_q8(Hq, Hkv, q_dtype):
    for seed in range(4):
        b = Batch(LENS, Hq, Hkv, seed=seed, q8=True, q_dtype=q_dtype)
        same = torch.from_numpy(_same(b.q.float().cpu().numpy())).cuda()
        assert same.float().mean() > 0.9
        ref, ref_lse = L.attn_decode_q8(*b.cache, b.q, b.bt, b.lens_t, want_lse=True)
        acc = torch.zeros(len(LENS), b.bt.shape[1] * 32, device="cuda")
        got = [L.attn_decode_window_q8(*b.cache, b.q, b.bt, b.lens_t, *w, want_lse=True)
               for w in ((3000, 0), (1, 3000), (2**31 - 1, 4))]
        got.append(L.attn_decode_weights_q8(*b.cache, b.q, b.bt, b.lens_t, acc, want_lse=True))
        L.check_status()
        for out, lse in got:
            assert torch.equal(out[same], ref[same]) and torch.equal(lse[same], ref_lse[same])


def test_the_two_scales_are_one_ulp_apart_at_most():
    """And a quantised integer differs only where a value lies on the border of two, by one."""
    rng = np.random.default_rng(0)
    q = rng.standard_normal((4000, 128)).astype(np.float16).astype(np.float32)
    (a, da), (b, db) = quantise_q8(q, product=True), quantise_q8(q)
    diff = np.abs(a.astype(int) - b.astype(int)).reshape(-1, 32).max(-1)
    assert diff.max() <= 1 and (diff > 0).mean() < 1e-3
    assert (np.abs(da.view(np.int16).astype(int) - db.view(np.int16)) <= 1).all()
