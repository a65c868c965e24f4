"""Rows with accumulated weights whose sequence is truncated or removed: what is appended afterwards starts
without weight and at its own position."""
import numpy as np
import pytest
import torch

import localstack_b200 as L
from tests.test_gpu_evict import select_ref

pytestmark = pytest.mark.gpu


def _append(pages, slot, n):
    pages.alloc(torch.tensor([slot], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda"), n)


def _check_select(w, pages, budget, n_sink, n_recent):
    state = [x.cpu().numpy() for x in (w.acc, w.pos, w.held, w.shift)]
    lens = pages.seq_lens.tolist()
    m = w.select(pages.seq_lens, budget, n_sink, n_recent)
    L.check_status()
    for b, (s, d) in enumerate(select_ref(*state, lens, budget, n_sink, n_recent)):
        assert m.src[b, :m.n[b]].tolist() == s and m.dst[b, :m.n[b]].tolist() == d
    return m


@pytest.mark.parametrize("side", [False, True])
def test_truncate_append_select(side):
    """A row that was never evicted from: cut to 100 keys, 150 appended. The new keys have no weight, so the
    eviction keeps the old ones (and the newest, protected), whatever stood behind the cut."""
    stream = torch.cuda.Stream() if side else None
    pages, w = L.DevicePages(2 * 320, 2, 10), L.KvWeights(2, 10)
    for slot in (0, 1):
        _append(pages, slot, 300)
    w.acc[:, :300] = torch.rand(2, 300, device="cuda") + 1.0
    other = w.acc[1].clone()
    torch.cuda.synchronize()
    w.release(pages, 0, 100, stream=stream)
    torch.cuda.synchronize()
    assert pages.seq_lens.tolist() == [100, 300]
    assert (w.acc[0, :100] >= 1).all() and not w.acc[0, 100:].any() and torch.equal(w.acc[1], other)
    _append(pages, 0, 150)
    budget, n_sink, n_recent = 120, 4, 10
    m = _check_select(w, pages, budget, n_sink, n_recent)
    # 110 kept keys besides the 10 recent ones: all of the 100 old ones and the first ten new ones
    assert m.n[0] == 10 and m.src[0, :10].tolist() == list(range(240, 250)) and m.dst[0, :10].tolist() == list(range(110, 120))
    w.finish(pages, m)
    L.check_status()
    assert w.pos[0, :budget].tolist() == list(range(110)) + list(range(240, 250)) and w.shift.tolist()[0] == 130


def test_after_an_eviction():
    """Tokens that came after the eviction can be taken back; a cut among the keys that it left is refused and
    changes nothing; the next tokens have the positions that were given up."""
    pages, w = L.DevicePages(320, 1, 10), L.KvWeights(1, 10)
    _append(pages, 0, 300)
    w.acc[0, :300] = torch.rand(300, device="cuda")
    w.finish(pages, _check_select(w, pages, 200, 4, 30))
    _append(pages, 0, 50)  # positions 300 .. 349 at indexes 200 .. 249
    w.acc[0, 200:250] = 5.0
    before = [x.clone() for x in (w.acc, w.pos, w.held, w.shift, pages.seq_lens, pages.free_top)]
    for keep in (1, 199):
        with pytest.raises(ValueError):
            w.release(pages, 0, keep)
    assert all(torch.equal(a, b) for a, b in zip(before, (w.acc, w.pos, w.held, w.shift, pages.seq_lens, pages.free_top)))
    w.release(pages, 0, 220)
    assert pages.seq_lens.tolist() == [220] and (w.acc[0, 200:220] == 5).all() and not w.acc[0, 220:].any()
    slot = torch.zeros(1, dtype=torch.int32, device="cuda")
    _, pos, _ = pages.alloc_step(slot)
    assert w.positions(pos, slot).tolist() == [320]
    _append(pages, 0, 39)
    w.acc[0, 220:260] = torch.rand(40, device="cuda")
    m = _check_select(w, pages, 200, 4, 30)
    w.finish(pages, m)
    L.check_status()
    at = w.pos[0, :200].tolist()
    assert len(set(at)) == 200 and set(at) >= set(range(4)) | set(range(330, 360)) and max(at) == 359
    w.release(pages, 0, 200)  # at held: nothing to drop
    assert pages.seq_lens.tolist() == [200] and w.pos[0, :200].tolist() == at
    w.release(pages, 0)
    L.check_status()
    assert not w.acc.any() and w.held.tolist() == w.shift.tolist() == pages.seq_lens.tolist() == [0]
    assert np.array_equal(np.sort(pages.free_list()), np.arange(10))
