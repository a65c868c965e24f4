"""Decode attention over a sliding window with sinks, against f64 (bounds: tests/bounded_ref.py)."""
import numpy as np
import pytest
import torch

import localstack_b200 as L
from localstack_b200 import _lib
from tests.bounded_ref import Batch, close, window_mask

pytestmark = pytest.mark.gpu

LENS = [0, 1, 31, 32, 33, 64, 100, 257, 1000]


def _run(b, window, n_sink, **kw):
    fn = L.attn_decode_window_q8 if b.q8 else L.attn_decode_window
    out, lse = fn(*b.cache, b.q, b.bt, b.lens_t, window, n_sink, want_lse=True, **kw)
    L.check_status()
    return out, lse


def _check(b, out, lse, window, n_sink):
    bf16 = out.dtype == torch.bfloat16
    out, lse = out.float().cpu().numpy(), lse.cpu().numpy()
    for i in range(len(b.lens)):
        o, l, _, t_o, t_l, _ = b.decode_ref(i, window, n_sink)
        close(out[i:i + 1], o, t_o, bf16, f"out of length {b.lens[i]}")
        close(lse[i:i + 1], l, t_l, False, f"lse of length {b.lens[i]}")


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (16, 3), (31, 4), (32, 32), (33, 33), (100, 70), (256, 64),
                                           (999, 1), (1000, 7), (5000, 4), (7, 5000), (2**31 - 1, 2**31 - 1)])
def test_windows_and_sinks(window, n_sink, q8):
    b = Batch(LENS, 32, 4, seed=window % 1000 + n_sink % 1000, q8=q8)
    out, lse = _run(b, window, n_sink)
    assert not out[0].any() and torch.isinf(lse[0]).all()  # no keys: zeros
    _check(b, out, lse, window, n_sink)


@pytest.mark.parametrize("Hq,Hkv", [(16, 8), (28, 4), (12, 2), (8, 1), (4, 4), (48, 12), (5, 5)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_dtype", [torch.float16, torch.float32])
def test_heads_and_types(Hq, Hkv, out_dtype, q_dtype):
    b = Batch([5, 700, 64, 333], Hq, Hkv, seed=Hq, q_dtype=q_dtype)
    out, lse = _run(b, 130, 9, out_dtype=out_dtype)
    assert out.dtype == out_dtype
    _check(b, out, lse, 130, 9)


@pytest.mark.parametrize("Hq,Hkv", [(16, 8), (28, 4), (12, 2), (20, 10)])
def test_heads_q8_bf16(Hq, Hkv):
    b = Batch([5, 700, 0, 333], Hq, Hkv, seed=Hq, q8=True)
    out, lse = _run(b, 130, 9, out_dtype=torch.bfloat16)
    _check(b, out, lse, 130, 9)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("lens", [[4000], [20000], [5000, 3, 17, 9000], list(range(1, 2000, 37))])
@pytest.mark.parametrize("n_ctas", [0, 1, 7, 300])
def test_splits(lens, n_ctas, q8):
    """One long sequence over many CTAs (the combine's paths), a few, and a batch merged by rows."""
    b = Batch(lens, 32, 4, seed=len(lens) + n_ctas, q8=q8)
    out, lse = _run(b, 1500, 40, n_ctas=n_ctas, out_dtype=torch.bfloat16)
    _check(b, out, lse, 1500, 40)


@pytest.mark.parametrize("q8", [False, True])
def test_hidden_cells_and_table_entries_do_not_matter(q8):
    """NaN and infinities in every cell outside the window and the sinks (inside the visible pages
    too), and page ids out of range in the gap: neither is looked at."""
    lens, window, n_sink = [500, 77, 33, 1200, 64], 45, 5
    b = Batch(lens, 16, 8, seed=3, q8=q8)
    want, want_lse = _run(b, window, n_sink)
    b.poison([np.flatnonzero(window_mask([n - 1], n, window, n_sink)[0]) for n in lens])
    for i, n in enumerate(lens):
        lo, hi = (n_sink + 31) // 32, max(0, n - window) // 32
        b.bt[i, lo:max(lo, hi)] = -7
        b.bt[i, (n + 31) // 32:] = 1 << 30
    got, lse = _run(b, window, n_sink)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    _check(b, got, lse, window, n_sink)


def test_a_window_over_everything_is_attn_decode():
    """The same page-groups in the same split: the same bits as the whole-sequence decode."""
    b = Batch(LENS + [3000], 32, 4, seed=5)
    ref, ref_lse = L.attn_decode(*b.cache, b.q, b.bt, b.lens_t, want_lse=True)
    for window, n_sink in ((3000, 0), (1, 3000), (2**31 - 1, 4)):
        out, lse = _run(b, window, n_sink)
        assert torch.equal(out, ref) and torch.equal(lse, ref_lse)


def test_bad_visible_page_and_length_are_reported():
    b = Batch([300, 40], 32, 4, seed=6)
    b.bt[0, 0] = 1 << 20  # the sinks' page
    out = L.attn_decode_window(*b.cache, b.q, b.bt, b.lens_t, 50, 4)
    with pytest.raises(L.LstkError) as e:
        L.check_status()
    assert e.value.code == _lib.LSTK_ERR_DEVICE_INDEX and torch.isfinite(out).all()
    b = Batch([300, 40], 32, 4, seed=6)
    b.lens_t[1] = 10 ** 6  # past the table: clamped to it
    L.attn_decode_window(*b.cache, b.q, b.bt, b.lens_t, 50, 4)
    with pytest.raises(L.LstkError):
        L.check_status()


def test_stream_graph_and_moving_lengths():
    """Captured once with the lengths on the device, replayed as the sequences grow, on a side stream,
    while another captured graph with a workspace of its own runs on the current one."""
    window, n_sink = 64, 4
    b = Batch([400, 90, 65], 32, 4, seed=8)
    c = Batch([800], 16, 8, seed=9)
    out, lse = torch.empty_like(b.q, dtype=torch.bfloat16), torch.empty(3, 32, device="cuda")
    out_c = torch.empty_like(c.q, dtype=torch.float32)
    ws, ws_c = L.DecodeWorkspace(3, 32, 4), L.DecodeWorkspace(1, 16, 8)
    call = lambda: L.attn_decode_window(*b.cache, b.q, b.bt, b.lens_t, window, n_sink, out=out, lse_out=lse,  # noqa: E731
                                        want_lse=True, workspace=ws)
    call_c = lambda: L.attn_decode_window(*c.cache, c.q, c.bt, c.lens_t, 99, 1, out=out_c, workspace=ws_c)  # noqa: E731
    call(), call_c()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs = []
    for f in (call, call_c):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            f()
        graphs.append(g)
    for lens in ([400, 90, 65], [33, 64, 1], [0, 70, 66]):
        b.lens = lens
        b.lens_t.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        L.check_status()
        _check(b, out, lse, window, n_sink)
        o, _, _, t, _, _ = c.decode_ref(0, 99, 1)
        close(out_c.cpu().numpy(), o, t)


def _policy(wait_ns, flag):
    _lib.check(L.lib().lstk_cuda_set_wait_policy(int(wait_ns), None if flag is None else flag.data_ptr()))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("op", ["window", "weights", "prefill"])
def test_a_wait_that_runs_out_is_reported_and_the_context_stays_usable(op, q8):
    """The loaders are gated on a flag that nothing sets, with a limit of 2 ms (host-visible status, no
    fault): LSTK_ERR_TIMEOUT, and the next call is right."""
    b = Batch([4000, 33, 1, 700], 32, 4, seed=12, q8=q8)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    acc = torch.zeros(4, b.bt.shape[1] * 32, device="cuda")
    sfx = "_q8" if q8 else ""

    def call():
        if op == "window":
            return getattr(L, "attn_decode_window" + sfx)(*b.cache, b.q, b.bt, b.lens_t, 300, 4)
        if op == "weights":
            return getattr(L, "attn_decode_weights" + sfx)(*b.cache, b.q, b.bt, b.lens_t, acc)
        return getattr(L, "attn_prefill_window" + sfx)(*b.cache, b.q, i32([0, 1, 2, 3, 4]), b.lens_t - 1, b.lens_t, b.bt, 1,
                                                       300, 4)

    want = call()
    L.check_status()
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    _policy(2_000_000, flag)
    try:
        call()
        with pytest.raises(L.LstkError) as e:
            L.check_status()
        assert e.value.code == _lib.LSTK_ERR_TIMEOUT
        flag.fill_(1)  # a gate that is open changes nothing
        _policy(500_000_000, flag)
        acc.zero_()
        assert torch.equal(call(), want)
        L.check_status()
    finally:
        _policy(0, None)
    acc.zero_()
    assert torch.equal(call(), want)
    L.check_status()


def test_streams_given_by_the_caller():
    """A call on another stream than the current one: its outputs and scratch belong to that stream, and the
    current stream and device are as before."""
    b = Batch([900, 64], 32, 4, seed=13, q_dtype=torch.float32)
    side = torch.cuda.Stream()
    acc, acc2 = (torch.zeros(2, b.bt.shape[1] * 32, device="cuda") for _ in range(2))
    start, pos0 = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), b.lens_t - 1
    torch.cuda.synchronize()
    results = []
    for stream in (None, side):
        before = torch.cuda.current_stream()
        results.append((L.attn_decode_window(*b.cache, b.q, b.bt, b.lens_t, 70, 3, stream=stream),
                        L.attn_decode_weights(*b.cache, b.q, b.bt, b.lens_t, acc if stream is None else acc2, stream=stream),
                        L.attn_prefill_window(*b.cache, b.q, start, pos0, b.lens_t, b.bt, 1, 70, 3, stream=stream)))
        assert torch.cuda.current_stream() == before and torch.cuda.current_device() == 0
        torch.cuda.synchronize()
    L.check_status()
    assert all(torch.equal(x, y) for x, y in zip(*results)) and torch.equal(acc, acc2)


def test_empty_calls():
    b = Batch([40], 16, 8, seed=14)
    none = lambda *shape, dtype=torch.int32: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    q, bt, lens = none(0, 16, 128, dtype=torch.float16), none(0, 2), none(0)
    out, lse = L.attn_decode_window(*b.cache, q, bt, lens, 5, want_lse=True)
    assert out.shape == (0, 16, 128) and lse.shape == (0, 16)
    assert L.attn_decode_weights(*b.cache, q, bt, lens, none(0, 64, dtype=torch.float32)).shape == (0, 16, 128)
    start = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert L.attn_prefill_window(*b.cache, q, start, lens, lens, bt, 0, 5).shape == (0, 16, 128)
    w = L.KvWeights(0, 2)
    m = w.select(lens, 40)
    L.kv_move(*b.cache, bt, m)
    L.check_status()


@pytest.mark.parametrize("op", ["window", "weights", "prefill", "move"])
def test_pages_past_32_bit_offsets(op):
    """A cache of 5 GB a side whose pages lie at its end: cells past 2^31 elements and bytes."""
    Hkv, n = 8, 100
    n_pages = (1 << 31) // (32 * Hkv * 128) + 8192  # 2^31 elements and 0.27 G more
    b = Batch([n], 16, Hkv, seed=15)
    big = [torch.empty(n_pages * 32, Hkv, 128, dtype=torch.float16, device="cuda") for _ in range(2)]
    pages = [n_pages - 1, n_pages - 17, 3, n_pages - 2]
    bt = torch.tensor([pages], dtype=torch.int32, device="cuda")
    for i, page in enumerate(pages):
        src = int(b.bt_host[0, i]) * 32
        for x, y in zip(big, b.cache):
            x[page * 32:(page + 1) * 32] = y[src:src + 32]
    start, pos0 = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([n - 1], dtype=torch.int32, device="cuda")
    if op == "move":
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        L.kv_move(*big, bt, L.KvMoves(i32([2]), i32([[97, 99]]), i32([[0, 40]]), 90))
        L.check_status()
        for x, y in zip(big, b.cache):
            c = b.cells(0)
            assert torch.equal(x[pages[0] * 32], y[int(c[97])]) and torch.equal(x[pages[1] * 32 + 8], y[int(c[99])])
        return
    if op == "window":
        got, want = (L.attn_decode_window(*c, b.q, t, b.lens_t, 50, 3) for c, t in ((big, bt), (b.cache, b.bt)))
    elif op == "weights":
        accs = [torch.zeros(1, 128, device="cuda") for _ in range(2)]
        got, want = (L.attn_decode_weights(*c, b.q, t, b.lens_t, a) for c, t, a in ((big, bt, accs[0]), (b.cache, b.bt, accs[1])))
        assert torch.equal(*accs)
    else:
        got, want = (L.attn_prefill_window(*c, b.q, start, pos0, b.lens_t, t, 1, 50, 3)
                     for c, t in ((big, bt), (b.cache, b.bt)))
    L.check_status()
    assert torch.equal(got, want)


def _poison_keys(b, at, head):
    """A NaN in KV head `head` of the key at(n) of every sequence but the last."""
    for i in range(len(b.lens) - 1):
        cell = b.cells(i)[at(b.lens[i])]
        (b.cache[0].d if b.q8 else b.cache[0])[cell, head] = float("nan")


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [[20, 300], [600, 300], [5000, 300], list(range(20, 900, 40))])
def test_a_nan_key_makes_the_rows_that_see_it_nan(lens, out_dtype, q8):
    """Whether one CTA has the whole row or pieces of it are merged; other heads and sequences are not touched."""
    b = Batch(lens, 16, 4, seed=1, q8=q8)
    _poison_keys(b, lambda n: n - 5, 2)
    out, lse = _run(b, 100000, 4, out_dtype=out_dtype)
    group = slice(8, 12)
    assert out[:-1, group].isnan().all() and lse[:-1, group].isnan().all()
    out[:-1, group] = 0
    lse[:-1, group] = 0
    assert not out.isnan().any() and not lse.isnan().any()
    out, lse = _run(b, 3, 4, out_dtype=out_dtype)  # out of the window
    _check(b, out, lse, 3, 4)
    b.q.fill_(float("nan"))
    if not q8:
        out, lse = _run(b, 100000, 4, out_dtype=out_dtype)
        assert out.isnan().all() and lse.isnan().all()


@pytest.mark.parametrize("Hq,Hkv", [(16, 8), (32, 4), (12, 12)])
@pytest.mark.parametrize("q8", [False, True])
def test_one_sequence_in_a_long_table(Hq, Hkv, q8):
    """Fewer pages than CTAs: some CTAs have none, and what earlier calls left in the workspace stays out."""
    ws = L.DecodeWorkspace(1, Hq, Hkv)
    ws.buf.fill_(0xff)  # NaN
    for n in (1, 32, 33, 64, 65, 100, 513, 1000, 2047, 2400, 4700, 0, 40):
        b = Batch([n], Hq, Hkv, seed=n, q8=q8)
        b.bt = torch.cat([b.bt, b.bt[:, :1].expand(1, 400)], 1)
        for window, n_sink, dtype in ((1 << 20, 0, torch.float32), (1024, 4, torch.bfloat16), (31, 1, torch.float32)):
            out, lse = _run(b, window, n_sink, out_dtype=dtype, workspace=ws)
            _check(b, out, lse, window, n_sink)
