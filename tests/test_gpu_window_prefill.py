"""Prefill attention over a sliding window with sinks, against f64 (bounds: tests/bounded_ref.py)."""
import numpy as np
import pytest
import torch

import localstack_b200 as L
from localstack_b200 import _lib
from tests.bounded_ref import Batch, attend, close, dequant, quantise_q8, vals, window_mask

pytestmark = pytest.mark.gpu


class Chunks:
    """Sequences of (first query position, query tokens, keys)."""

    def __init__(self, seqs, Hq, Hkv, seed=0, q8=False, q_dtype=torch.float16, spare_rows=0):
        self.seqs = seqs
        T = sum(t for _, t, _ in seqs)
        self.b = Batch([n for _, _, n in seqs], Hq, Hkv, seed=seed, q8=q8, q_dtype=q_dtype, n_q=T + spare_rows)
        b = self.b
        if q8:  # the prefill of a q8_0 cache reads d * q rounded to f16, and f16 queries
            planes = [quantise_q8(vals(x)) for x in (b.kb, b.vb)]
            b.k_host, b.v_host = (dequant(*p).astype(np.float16).astype(np.float64) for p in planes)
            b.q_host = b.q.half().cpu().numpy().astype(np.float64)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        self.starts = np.concatenate([[0], np.cumsum([t for _, t, _ in seqs])])
        self.start_t, self.pos0_t = i32(self.starts.tolist()), i32([p for p, _, _ in seqs])
        self.max_q = max(t for _, t, _ in seqs)

    def run(self, window, n_sink, **kw):
        b = self.b
        fn = L.attn_prefill_window_q8 if b.q8 else L.attn_prefill_window
        out = fn(*b.cache, b.q, self.start_t, self.pos0_t, b.lens_t, b.bt, self.max_q, window, n_sink, **kw)
        L.check_status()
        return out

    def check(self, out, window, n_sink):
        b, bf16 = self.b, out.dtype == torch.bfloat16
        out = out.float().cpu().numpy()
        for i, (p0, t, n) in enumerate(self.seqs):
            rows = slice(self.starts[i], self.starts[i + 1])
            c = b.cells(i)
            seen = window_mask(p0 + np.arange(t), n, window, n_sink)
            o, _, _, tol, _, _ = attend(b.q_host[rows], b.k_host[c], b.v_host[c], seen, prefill=True)
            close(out[rows], o, tol, bf16, f"out of sequence {i}")


RAGGED = [(0, 1, 1), (0, 70, 70), (31, 2, 33), (500, 129, 629), (0, 0, 5), (64, 64, 128), (1000, 17, 1017)]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (16, 5), (32, 32), (33, 4), (100, 70), (128, 0), (300, 64),
                                           (5000, 4), (7, 5000), (2**31 - 1, 2**31 - 1)])
def test_windows_and_sinks(window, n_sink, q8):
    c = Chunks(RAGGED, 8, 2, seed=window % 1000 + n_sink % 1000, q8=q8)
    c.check(c.run(window, n_sink), window, n_sink)


@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (8, 4), (32, 4), (16, 8), (8, 1)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_dtype", [torch.float16, torch.float32])
def test_heads_and_types(Hq, Hkv, out_dtype, q_dtype):
    c = Chunks([(300, 200, 500), (0, 77, 77)], Hq, Hkv, seed=Hq, q_dtype=q_dtype)
    out = c.run(90, 5, out_dtype=out_dtype)
    assert out.dtype == out_dtype
    c.check(out, 90, 5)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_many_tiles_and_items(out_dtype):
    """More items than SMs, windows of several tiles, sinks across pages."""
    c = Chunks([(0, 1500, 1500), (2000, 700, 2700), (0, 333, 333)], 16, 8, seed=3)
    c.check(c.run(640, 50, out_dtype=out_dtype), 640, 50)


def test_more_sequences_than_the_schedule_sorts():
    """150 short sequences (some without queries or keys), taken in their own order."""
    rng = np.random.default_rng(4)
    seqs = []
    for i in range(150):
        t = int(rng.integers(0, 40))
        seqs.append((int(rng.integers(0, 90)), t, 0)) if i % 29 == 5 else seqs.append((n := int(rng.integers(0, 90)), t, n + t))
    for window, n_sink in ((33, 4), (500, 0)):
        c = Chunks(seqs, 8, 2, seed=9)
        c.check(c.run(window, n_sink, out_dtype=torch.bfloat16), window, n_sink)


@pytest.mark.parametrize("T", [1, 16, 33, 64, 65, 300])
def test_one_sequence(T):
    for p0 in (0, 777):
        c = Chunks([(p0, T, p0 + T)], 16, 8, seed=T)
        c.check(c.run(100, 5), 100, 5)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("seqs,Hq,Hkv", [([(4999, 1, 5000)], 8, 8), ([(4000, 3, 4003), (100, 2, 102), (0, 0, 9)], 8, 2),
                                         ([(2900, 70, 2970)], 32, 4), ([(9, 1, 10)] * 5 + [(3000, 1, 3001)], 16, 8)])
def test_few_queries_behind_long_contexts(seqs, Hq, Hkv, q8):
    """Split along the keys (a workspace that allows it), and not (none): both within the bounds of the exact
    result, rows of no sequence left alone."""
    T = sum(t for _, t, _ in seqs)
    for window, n_sink, dtype in ((5000, 0, torch.float32), (1999, 33, torch.bfloat16), (2**31 - 1, 4, torch.float32)):
        c = Chunks(seqs, Hq, Hkv, seed=T, q8=q8, spare_rows=2)
        need = L.prefill_window_workspace_bytes(c.b.q, Hkv, c.max_q, c.b.bt, window, n_sink)
        assert need > 0
        for ws in (torch.full((need,), 0xff, dtype=torch.uint8, device="cuda"), torch.empty(256, dtype=torch.uint8, device="cuda")):
            out = torch.full((T + 2, Hq, 128), 7.0, dtype=dtype, device="cuda")
            c.run(window, n_sink, out=out, workspace=ws)
            c.check(out[:T], window, n_sink)
            assert (out[T:] == 7).all()


def test_rows_that_see_nothing_and_rows_of_no_sequence():
    """Keys end before some queries' windows begin: those rows are zeros; spare rows are left alone."""
    seqs = [(100, 100, 120), (500, 40, 100), (10, 30, 0)]
    for out_dtype in (torch.float32, torch.bfloat16):
        c = Chunks(seqs, 8, 2, seed=4, spare_rows=9)
        out = torch.full((179, 8, 128), 7.0, dtype=out_dtype, device="cuda")
        c.run(20, 0, out=out)
        c.check(out[:170], 20, 0)
        assert not out[40:170].any() and (out[170:] == 7).all()
        assert out[:39].float().abs().sum((1, 2)).min() > 0
        c.check(c.run(20, 3, out_dtype=out_dtype)[:170], 20, 3)


def test_a_window_over_everything_is_attn_prefill():
    """The two kernels take the row maxima over different key sets, so their roundings differ: both are
    held to the exact result's bound, and hence to twice that bound of one another."""
    c = Chunks(RAGGED, 8, 2, seed=5)
    b = c.b
    c.check(L.attn_prefill(*b.cache, b.q, c.start_t, c.pos0_t, b.lens_t, b.bt, c.max_q), 1017, 0)
    c.check(c.run(1017, 0), 1017, 0)
    assert torch.equal(c.run(1017, 0), c.run(2**31 - 1, 6))  # the same keys in the same tiles


@pytest.mark.parametrize("q8", [False, True])
def test_hidden_cells_and_table_entries_do_not_matter(q8):
    """NaN and infinities in every cell that no query of the sequence sees, one query tile each (G = 4:
    32 tokens), and page ids out of range in the gap."""
    seqs = [(500, 30, 530), (77, 1, 78), (10, 20, 30), (320, 32, 340)]
    window, n_sink = 45, 5
    c = Chunks(seqs, 8, 2, seed=6, q8=q8)
    b = c.b
    want = c.run(window, n_sink)
    b.poison([np.flatnonzero(window_mask(p0 + np.arange(t), n, window, n_sink).any(0)) for p0, t, n in seqs])
    for i, (p0, t, n) in enumerate(seqs):
        lo, hi = (n_sink + 31) // 32, max(0, p0 + 1 - window) // 32
        b.bt[i, lo:max(lo, hi)] = -7
        b.bt[i, (n + 31) // 32:] = 1 << 30
    got = c.run(window, n_sink)
    assert torch.equal(got, want)
    c.check(got, window, n_sink)


def test_bad_page_and_rows_are_reported():
    c = Chunks([(300, 64, 364), (0, 20, 20)], 8, 2, seed=7)
    c.b.bt[0, 10] = 1 << 20
    with pytest.raises(L.LstkError) as e:
        c.run(60, 4)
    assert e.value.code == _lib.LSTK_ERR_DEVICE_INDEX
    c = Chunks([(300, 64, 364), (0, 20, 20)], 8, 2, seed=7)
    c.start_t[2] = 1000  # rows behind the last one: the sequence is skipped
    with pytest.raises(L.LstkError):
        c.run(60, 4)


def test_graph_on_another_stream():
    c = Chunks([(0, 100, 100), (200, 30, 230)], 8, 2, seed=8, q_dtype=torch.float32)
    b = c.b
    out = torch.empty_like(b.q, dtype=torch.bfloat16)
    ws = torch.empty(max(b.q.numel() * 2 + 256, L.prefill_window_workspace_bytes(b.q, 2, c.max_q, b.bt, 40, 3)),
                     dtype=torch.uint8, device="cuda")
    c.run(40, 3, out=out, workspace=ws)
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        L.attn_prefill_window(*b.cache, b.q, c.start_t, c.pos0_t, b.lens_t, b.bt, c.max_q, 40, 3, out=out, workspace=ws)
    c.seqs = [(0, 100, 100), (150, 30, 180)]
    c.pos0_t.copy_(torch.tensor([0, 150], dtype=torch.int32))
    b.lens_t.copy_(torch.tensor([100, 180], dtype=torch.int32))
    out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        g.replay()
    torch.cuda.synchronize()
    L.check_status()
    b.lens = [100, 180]
    c.check(out, 40, 3)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("seqs,window", [([(100, 140, 240)], 60), ([(0, 300, 300), (30, 90, 120)], 60),
                                         ([(4990, 10, 5000)], 100000), ([(4970, 30, 5000), (100, 40, 140)], 4000)])
def test_a_nan_key_makes_the_rows_that_see_it_nan(seqs, window, out_dtype, q8):
    c = Chunks(seqs, 16, 4, seed=2, q8=q8)
    b = c.b
    at = [max(n - 120, 3) for _, _, n in seqs]
    for i in range(len(seqs)):
        (b.cache[0].d if q8 else b.cache[0])[b.cells(i)[at[i]], 2] = float("nan")
    out = c.run(window, 2, out_dtype=out_dtype)
    for i, (p0, t, n) in enumerate(seqs):
        sees = torch.from_numpy(window_mask(p0 + np.arange(t), n, window, 2)[:, at[i]]).cuda()
        o = out[c.starts[i]:c.starts[i + 1]]
        assert torch.equal(o.isnan().all(-1), sees[:, None] & (torch.arange(16, device="cuda") // 4 == 2))
        assert torch.equal(o.isnan().any(-1), o.isnan().all(-1))


@pytest.mark.parametrize("q8", [False, True])
def test_positions_at_the_ends_of_32_bits(q8):
    """First positions close to 2^31 - 1 (later ones pass it) and below zero (those queries see no key)."""
    seqs = [(2**31 - 5, 40, 100), (2**31 - 1, 300, 260), (-7, 30, 100), (-(2**31), 3, 10)]
    c = Chunks(seqs, 8, 2, seed=3, q8=q8)
    for window, n_sink in ((2**31 - 1, 0), (2**31 - 10, 5), (50, 3)):
        c.check(c.run(window, n_sink), window, n_sink)


@pytest.mark.parametrize("n,longest", [(129, 400), (300, 700), (200, 3)])
@pytest.mark.parametrize("q8", [False, True])
def test_many_sequences_of_uneven_lengths(n, longest, q8):
    """More sequences than are sorted, most of one query or none, a few of several pairs, and one whose rows are
    bad (the others are computed all the same)."""
    rng = np.random.default_rng(n)
    seqs = []
    for i in range(n):
        t = longest if i % 67 == 31 else int(rng.integers(0, 3))
        p0 = int(rng.integers(0, 200))
        seqs.append((p0, t, 0 if i % 29 == 5 else p0 + t))
    c = Chunks(seqs, 8, 4, seed=9, q8=q8)
    for window, n_sink in ((33, 4), (500, 0)):
        c.check(c.run(window, n_sink, out_dtype=torch.bfloat16), window, n_sink)
    want = c.run(90, 2)
    a, b = int(c.starts[n - 1]), int(c.starts[n])
    c.start_t[n] = 1 << 30
    out = torch.zeros_like(want)
    with pytest.raises(L.LstkError):
        c.run(90, 2, out=out)
    assert torch.equal(out[:a], want[:a]) and not out[a:b].any()
