"""Eviction by accumulated weight: the selection, the moves and the bookkeeping against numpy restatements
(whole numbers and moved bytes: equal), and a serving loop that runs past its budget."""
import numpy as np
import pytest
import torch

import localstack_b200 as L
from localstack_b200 import _lib
from localstack_b200.kv_cache import KvCache
from oracle import oracle as O
from tests.bounded_ref import attend, close, vals

pytestmark = pytest.mark.gpu


def select_ref(acc, pos, held, shift, lens, budget, n_sink, n_recent):
    """Per row the moves (src, dst lists)."""
    moves = []
    for b, n in enumerate(lens):
        if n <= budget:
            moves.append(([], []))
            continue
        i = np.arange(n, dtype=np.int64)
        at = np.where(i < held[b], pos[b, :n], i + int(shift[b]))
        safe = (at < n_sink) | (at >= n + int(shift[b]) - n_recent)
        a = np.where(np.isnan(acc[b, :n]), -np.inf, acc[b, :n]).astype(np.float64)
        nan = np.isnan(acc[b, :n]) & ~safe
        order = np.lexsort((i, np.where(safe, 0.0, -a), nan, ~safe))  # protected, not NaN, larger acc, lower index
        kept = np.zeros(n, bool)
        kept[order[:budget]] = True
        moves.append(((np.flatnonzero(kept[budget:]) + budget).tolist(), np.flatnonzero(~kept[:budget]).tolist()))
    return moves


def _state(rng, lens, cells, budget, ties=False, fresh=False):
    """Accumulated weights (zero behind the rows), a shuffled record of positions for the first keys."""
    B = len(lens)
    acc = np.exp(rng.standard_normal((B, cells)) * 2.5 - 4).astype(np.float32)
    if ties:
        acc = rng.integers(0, 3, (B, cells)).astype(np.float32) * np.float32(0.25)
    pos = rng.integers(0, 1 << 30, (B, cells)).astype(np.int32)
    held, shift = np.zeros(B, np.int32), np.zeros(B, np.int32)
    for b, n in enumerate(lens):
        acc[b, n:] = 0
        if not fresh:
            held[b], shift[b] = min(n, budget), rng.integers(0, 5000)
            r = rng.permutation(held[b])
            pos[b, :held[b]] = np.where(r < 3, r, r + shift[b])
    return acc, pos, held, shift


def _weights(state):
    return L.KvWeights.from_tensors(*(torch.from_numpy(x).cuda() for x in state))


def _check_select(w, state, lens, budget, n_sink, n_recent):
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    m = w.select(lens_t, budget, n_sink, n_recent)
    L.check_status()
    n, src, dst = (x.cpu().numpy() for x in (m.n, m.src, m.dst))
    for b, (s, d) in enumerate(select_ref(*state, lens, budget, n_sink, n_recent)):
        assert len(s) == len(d) == n[b], (b, len(s), n[b])
        assert src[b, :n[b]].tolist() == s and dst[b, :n[b]].tolist() == d
        assert (src[b, n[b]:] == -1).all() and (dst[b, n[b]:] == -1).all()
    return m


@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("budget,n_sink,n_recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (31, 4, 5), (32, 0, 32), (33, 33, 0),
                                                    (100, 4, 64), (500, 0, 0), (1000, 4, 200)])
def test_select(budget, n_sink, n_recent, ties, fresh):
    rng = np.random.default_rng(budget + n_sink)
    lens = [0, 1, 31, 32, 33, budget, budget + 1, budget + 63, 1100, 1500]
    state = _state(rng, lens, 1504, budget, ties, fresh)
    _check_select(_weights(state), state, lens, budget, n_sink, n_recent)


@pytest.mark.parametrize("cells,lens,budget", [(4096, [4096, 4000], 2000), (4128, [4128, 17], 4096),
                                               (16416, [16416, 9000, 16400], 8192), (32768, [32768, 32767], 31000),
                                               (300000, [299999, 1000], 4096), (300032, [300032], 299000)])
@pytest.mark.parametrize("ties", [False, True])
def test_select_long_rows(cells, lens, budget, ties):
    """Rows over clusters of 1 to 8 CTAs, and shares longer than the keys held in shared memory."""
    rng = np.random.default_rng(cells)
    state = _state(rng, lens, cells, budget, ties)
    _check_select(_weights(state), state, lens, budget, 33, 1000)


def test_select_special_values():
    """NaN (either sign) ranks lowest, -0 equals +0, infinities and subnormals keep their order, and
    protected tokens stay whatever their weight."""
    rng = np.random.default_rng(5)
    special = np.array([np.nan, -np.nan, 0.0, -0.0, np.inf, -np.inf, 1e-42, -1e-42, 1.0, -1.0, 3e38], np.float32)
    acc = special[rng.integers(0, special.size, (4, 320))]
    pos, held, shift = np.zeros((4, 320), np.int32), np.zeros(4, np.int32), np.array([0, 7, 0, 3], np.int32)
    state = (acc, pos, held, shift)
    for budget in (1, 60, 150, 319):
        _check_select(_weights(state), state, [320, 320, 300, 161], budget, 0, 0)
        _check_select(_weights(state), state, [320, 320, 300, 161], budget, min(9, budget // 2), budget // 3)
    acc[:] = np.nan
    _check_select(_weights(state), state, [320, 320, 300, 161], 60, 3, 10)
    acc[:] = 0
    _check_select(_weights(state), state, [320, 320, 300, 161], 60, 3, 10)


def test_select_reports_a_bad_length_and_repeats():
    rng = np.random.default_rng(6)
    lens = [300, 200]
    state = _state(rng, lens, 320, 100)
    w = _weights(state)
    m = _check_select(w, state, lens, 100, 4, 10)
    first = [x.clone() for x in (m.n, m.src, m.dst)]
    w.select(torch.tensor(lens, dtype=torch.int32, device="cuda"), 100, 4, 10, moves=m)
    assert all(torch.equal(a, b) for a, b in zip(first, (m.n, m.src, m.dst)))
    for bad in (-1, 321, 2**31 - 1):
        m = w.select(torch.tensor([300, bad], dtype=torch.int32, device="cuda"), 100, 4, 10)
        with pytest.raises(L.LstkError) as e:
            L.check_status()
        assert e.value.code == _lib.LSTK_ERR_DEVICE_INDEX
        assert m.n.tolist()[1] == 0 and torch.equal(m.src[0], first[1][0])


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("Hkv", [1, 2, 3, 4, 8, 12])
def test_move(Hkv, q8):
    rng = np.random.default_rng(Hkv)
    n_pages, max_blocks, n_cells = 40, 12, 40 * 32
    bt = rng.permutation(n_pages)[:36].reshape(3, max_blocks).astype(np.int32)
    cell = lambda b, i: bt[b, i // 32] * 32 + i % 32  # noqa: E731
    if q8:
        planes = [rng.integers(-128, 128, (n_cells, Hkv, 128)).astype(np.int8) if i % 2 == 0 else
                  rng.integers(0, 1 << 15, (n_cells, Hkv, 4)).astype(np.int16) for i in range(4)]
    else:
        planes = [rng.integers(-2**15, 2**15, (n_cells, Hkv, 128)).astype(np.int16) for _ in range(2)]
    t = [torch.from_numpy(p).cuda() for p in planes]
    t = [x.view(torch.float16) if x.dtype == torch.int16 else x for x in t]
    cache = (L.Q8Cache.from_planes(t[0], t[1]), L.Q8Cache.from_planes(t[2], t[3])) if q8 else tuple(t)
    budget, counts = 200, [57, 0, 150]
    src, dst = np.full((3, 160), -1, np.int32), np.full((3, 160), -1, np.int32)
    want = [p.copy() for p in planes]
    for b, k in enumerate(counts):
        src[b, :k] = np.sort(rng.permutation(np.arange(budget, 384))[:k])
        dst[b, :k] = np.sort(rng.permutation(budget)[:k])
        for p, o in zip(want, planes):
            p[cell(b, dst[b, :k])] = o[cell(b, src[b, :k])]
    m = L.KvMoves(*(torch.from_numpy(x).cuda() for x in (np.array(counts, np.int32), src, dst)), budget)
    run = lambda: (L.kv_move_q8 if q8 else L.kv_move)(*cache, torch.from_numpy(bt).cuda(), m)  # noqa: E731
    run()
    run()  # the sources stay, so a second time changes nothing
    L.check_status()
    for x, p in zip(t, want):
        assert np.array_equal((x.view(torch.int16) if x.dtype == torch.float16 else x).cpu().numpy(), p)


def test_move_skips_what_is_out_of_range():
    kc, vc = L.alloc_cache(64, 2), L.alloc_cache(64, 2)
    kc.copy_(torch.randn(64, 2, 128))
    before = kc.clone()
    bt = torch.tensor([[0, 9], [-1, 1]], dtype=torch.int32, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for src, dst in (([[40], [40]], [[1], [1]]), ([[64], [-1]], [[0], [32]])):
        L.kv_move(kc, vc, bt, L.KvMoves(i32([1, 1]), i32(src), i32(dst), 32))
        with pytest.raises(L.LstkError) as e:
            L.check_status()
        assert e.value.code == _lib.LSTK_ERR_DEVICE_INDEX and torch.equal(kc, before)


@pytest.mark.parametrize("n_slots", [1, 5, 1500])
def test_finish(n_slots):
    """acc, pos, held and shift of every row, and the pages against the host's KvCache truncating the rows
    in order."""
    rng = np.random.default_rng(n_slots)
    max_blocks, budget, n_sink, n_recent = (9, 100, 4, 20) if n_slots < 100 else (3, 40, 1, 7)
    cells = max_blocks * 32
    size = n_slots * cells
    lens = rng.integers(0, cells + 1, n_slots)
    lens[0] = cells
    pages = L.DevicePages(size, n_slots, max_blocks)
    host = KvCache(size)
    order = rng.permutation(n_slots)
    for part in (0, 1):  # scattered tables
        for b in order:
            n = int(lens[b])
            if (n // 2, n - n // 2)[part]:
                host.alloc(int(b), (n // 2, n - n // 2)[part])
    # the device starts from the host's state
    bt, hl = host.block_tables(np.arange(n_slots), max_blocks)
    pages.block_tables.copy_(torch.from_numpy(np.maximum(bt, 0)))
    assert np.array_equal(hl, lens)
    fl = host.free_blocks()
    pages.free_blocks[:fl.size] = torch.from_numpy(fl.view(np.int32)).cuda()
    pages.free_top.fill_(fl.size)
    pages.seq_lens.copy_(torch.from_numpy(hl))
    state = _state(rng, lens.tolist(), cells, budget)
    w = _weights(state)
    acc, pos, held, shift = (x.copy() for x in state)
    m = w.select(pages.seq_lens, budget, n_sink, n_recent)
    w.finish(pages, m)
    L.check_status()
    for b, (s, d) in enumerate(select_ref(*state, lens.tolist(), budget, n_sink, n_recent)):
        n = lens[b]
        if n <= budget:
            continue
        true = np.where(np.arange(n) < held[b], pos[b, :n], np.arange(n) + shift[b])
        pos[b, :budget] = true[:budget]
        pos[b, d], acc[b, d] = true[s], acc[b, s]
        acc[b, budget:n] = 0
        held[b], shift[b] = budget, shift[b] + n - budget
        host.truncate_seq(b, budget)
    assert np.array_equal(w.acc.cpu().numpy(), acc)
    got = w.pos.cpu().numpy()
    for b in range(n_slots):
        assert np.array_equal(got[b, :held[b]], pos[b, :held[b]])
    assert np.array_equal(w.held.cpu().numpy(), held) and np.array_equal(w.shift.cpu().numpy(), shift)
    assert np.array_equal(pages.free_list(), host.free_blocks())
    assert np.array_equal(pages.seq_lens.cpu().numpy(), np.minimum(lens, budget))
    assert int(pages.used_hwm.item()) == host.used_hwm


def test_finish_skips_moves_of_other_rows():
    rng = np.random.default_rng(9)
    state = _state(rng, [320], 320, 100)
    pages = L.DevicePages(320, 1, 10)
    pages.alloc(torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([320], dtype=torch.int32, device="cuda"), 320)
    w = _weights(state)
    m = w.select(pages.seq_lens, 100)
    m.src[0, 0], m.dst[0, 1] = 5, 100
    w.finish(pages, m)
    with pytest.raises(L.LstkError) as e:
        L.check_status()
    assert e.value.code == _lib.LSTK_ERR_DEVICE_INDEX and int(pages.seq_lens[0]) == 100


def test_refusals():
    w = L.KvWeights(2, 4)
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    for budget, sink, recent in ((0, 0, 0), (-1, 0, 0), (10, 11, 0), (10, 6, 5), (10, -1, 0), (10, 0, -1),
                                 (2**31 - 1, 2**31 - 1, 1)):
        with pytest.raises(L.LstkError):
            w.select(lens, budget, sink, recent)
    with pytest.raises(ValueError):
        w.select(lens.long(), 10)
    with pytest.raises(ValueError):
        w.select(lens[:1], 10)
    m = w.select(lens, 120)
    with pytest.raises(ValueError):
        w.select(lens, 64, moves=m)  # 64 moves a row do not fit in 8
    assert w.select(lens, 128).src.shape == (2, 0) and w.select(lens, 5000).n.tolist() == [0, 0]
    pages = L.DevicePages(256, 3, 4)
    with pytest.raises(L.LstkError):
        w.finish(pages, m)  # not the slots' rows
    with pytest.raises(L.LstkError):
        L.KvWeights(2, 3).finish(L.DevicePages(256, 2, 4), L.KvWeights(2, 3).select(lens, 10))
    with pytest.raises(ValueError):
        L.KvWeights.from_tensors(w.acc, w.pos.long(), w.held, w.shift)
    with pytest.raises(ValueError):
        L.kv_move(L.alloc_cache(64, 2), L.alloc_cache(64, 2), pages.block_tables, m)
    L.check_status()


@pytest.mark.parametrize("graph", [False, True])
def test_serving_past_the_budget(graph):
    """Three sequences decode 195 tokens each with 96 keys of budget: allocate, append (RoPE at the true
    positions), attend with accumulated weights, and evict 32 keys whenever a row reaches 128. Every
    step's output and weights against f64 attention over the tokens that the evictions left, every
    eviction against its restatement, the pages against the host's KvCache. With `graph`, the step and
    the eviction replay from CUDA graphs."""
    Hq, Hkv, budget, full, n_sink, n_recent, steps = 8, 2, 96, 128, 4, 20, 195
    B, max_blocks, layers = 3, 4, 2
    rng = np.random.default_rng(11)
    pages, host = L.DevicePages(B * full, B, max_blocks), KvCache(B * full)
    caches = [(L.alloc_cache(B * full, Hkv), L.alloc_cache(B * full, Hkv)) for _ in range(layers)]
    w, rope = L.KvWeights(B, max_blocks), L.rope_table(steps)
    slots = torch.arange(B, dtype=torch.int32, device="cuda")
    q_in, k_in, v_in = (torch.empty(layers, B, h, 128, device="cuda") for h in (Hq, Hkv, Hkv))
    outs = torch.empty(layers, B, Hq, 128, device="cuda")
    q16 = torch.empty(layers, B, Hq, 128, dtype=torch.float16, device="cuda")
    ws = L.WeightsWorkspace(B, Hq, Hkv, full)
    cells = torch.empty(B, dtype=torch.int64, device="cuda")
    pos, true_pos = (torch.empty(B, dtype=torch.int32, device="cuda") for _ in range(2))
    ok = torch.empty(B, dtype=torch.int32, device="cuda")
    moves = w.select(pages.seq_lens, budget, n_sink, n_recent)

    def step():
        pages.alloc_step(slots, cells, pos, ok)
        torch.add(pos, w.shift, out=true_pos)
        for l, (k, v) in enumerate(caches):
            L.kv_append(k, v, q_in[l], k_in[l], v_in[l], true_pos, cells, rope, q_out=q16[l])
            L.attn_decode_weights(k, v, q16[l], pages.block_tables, pages.seq_lens, w.acc, workspace=ws, out=outs[l])

    def evict():
        w.select(pages.seq_lens, budget, n_sink, n_recent, moves=moves)
        for k, v in caches:
            L.kv_move(k, v, pages.block_tables, moves)
        w.finish(pages, moves)

    if graph:
        side = torch.cuda.Stream()
        run = []
        for f in (step, evict):
            g = torch.cuda.CUDAGraph()
            if f is step:  # first uses happen outside a capture, on state that is put back
                saved = [x.clone() for x in (pages.free_blocks, pages.free_top, pages.block_tables, pages.seq_lens)]
                step(), evict()
                for x, y in zip((pages.free_blocks, pages.free_top, pages.block_tables, pages.seq_lens), saved):
                    x.copy_(y)
                w.acc.zero_(), pages.used_hwm.zero_()
                torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=side):
                f()
            run.append(g.replay)
        step, evict = run

    tokens = [[] for _ in range(B)]  # per slot: dict(pos, k, v per layer, acc), in index order
    for t in range(steps):
        ins = [rng.standard_normal((layers, B, h, 128)).astype(np.float32) for h in (Hq, Hkv, Hkv)]
        for x, a in zip((q_in, k_in, v_in), ins):
            x.copy_(torch.from_numpy(a))
        torch.cuda.synchronize()
        step()
        torch.cuda.synchronize()
        L.check_status()
        assert ok.tolist() == [1] * B and true_pos.tolist() == [t] * B
        for b in range(B):
            host.alloc(b, 1)
        scratch = [[np.zeros((32, Hkv, 128), np.uint16) for _ in range(2)] for _ in range(layers)]
        for b in range(B):
            tokens[b].append(dict(pos=t, acc=0.0, tol=0.0, k=[], v=[]))
        for l in range(layers):
            q_ref = O.kv_append(*(x[l] for x in ins), np.full(B, t, np.int32), np.arange(B, dtype=np.int64),
                                *scratch[l], None, None, 1e-6, 1e6)
            q_ref = q_ref.astype(np.float16).astype(np.float64)
            for b in range(B):
                tk = tokens[b]
                tk[-1]["k"].append(vals(scratch[l][0][b])), tk[-1]["v"].append(vals(scratch[l][1][b]))
                k, v = (np.stack([x[n][l] for x in tk]) for n in "kv")
                o, _, wt, tol, _, t_w = attend(q_ref[b:b + 1], k, v, np.ones((1, len(tk)), bool))
                close(outs[l, b:b + 1].cpu().numpy(), o, tol, what=f"step {t} layer {l} slot {b}")
                for x, a, e in zip(tk, wt, t_w):
                    x["acc"] += a
                    x["tol"] += e + (Hq + 1) * 2.0 ** -24 * x["acc"]
        acc = w.acc.cpu().numpy()
        for b in range(B):
            n = len(tokens[b])
            close(acc[b, :n], np.array([x["acc"] for x in tokens[b]]), np.array([x["tol"] for x in tokens[b]]),
                  what=f"weights at step {t}")
            assert not acc[b, n:].any()
        if len(tokens[0]) == full:
            state = [x.cpu().numpy() for x in (w.acc, w.pos, w.held, w.shift)]
            evict()
            torch.cuda.synchronize()
            L.check_status()
            for b, (s, d) in enumerate(select_ref(*state, [full] * B, budget, n_sink, n_recent)):
                for i, j in zip(s, d):
                    tokens[b][j] = tokens[b][i]
                del tokens[b][budget:]
                host.truncate_seq(b, budget)
                at = [x["pos"] for x in tokens[b]]
                assert set(at) >= set(range(n_sink)) | set(range(t + 1 - n_recent, t + 1)) and len(set(at)) == budget
                assert w.pos[b, :budget].tolist() == at
        assert np.array_equal(pages.free_list(), host.free_blocks())
        bt, hl = host.block_tables(np.arange(B), max_blocks)
        assert pages.seq_lens.tolist() == hl.tolist()
    assert w.shift.tolist() == [3 * (full - budget)] * B and w.positions(pos, slots).tolist() == [steps - 1] * B
    w.reset(1)
    assert not w.acc[1].any() and w.shift.tolist()[1] == 0 == w.held.tolist()[1] and w.acc[0].any()
