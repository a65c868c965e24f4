"""The bounded-cache entry points refuse bad arguments with the documented codes before touching a GPU."""
import ctypes

import pytest
import torch

import localstack_b200 as L
from localstack_b200 import _lib

F32, F16, BF16 = _lib.DTYPE_F32, _lib.DTYPE_F16, _lib.DTYPE_BF16
ARG, CAP, UNSUP = _lib.LSTK_ERR_INVALID_ARG, _lib.LSTK_ERR_CAPACITY, _lib.LSTK_ERR_UNSUPPORTED
P = 0x10000  # never dereferenced: validation fails first
BIG = 1 << 40


def _layout(hkv=8, hd=128, bs=32, n_cells=64):
    return ctypes.byref(_lib.KvLayout(n_cells, hkv, hd, bs))


def _caches(q8, bad):
    return ([None if bad == "k" else P, P] + ([P, P] if q8 else []))


def _window(q8=False, lay=None, bad="", q=P, qd=F16, B=1, Hq=16, bt=P, mb=4, lens=P, mx=0, window=10, sink=2, out=P,
            od=BF16, ws=P, wsb=BIG):
    fn = L.lib().lstk_cuda_attn_decode_window_q8 if q8 else L.lib().lstk_cuda_attn_decode_window
    return fn(lay or _layout(), *_caches(q8, bad), q, qd, B, Hq, bt, mb, lens, mx, window, sink, 0.1, out, od, None, ws,
              wsb, 0, None)


def _weights(q8=False, lay=None, bad="", q=P, qd=F16, B=1, Hq=16, bt=P, mb=4, lens=P, mx=0, acc=P, stride=128, out=P,
             od=F32, ws=P, wsb=BIG):
    fn = L.lib().lstk_cuda_attn_decode_weights_q8 if q8 else L.lib().lstk_cuda_attn_decode_weights
    return fn(lay or _layout(), *_caches(q8, bad), q, qd, B, Hq, bt, mb, lens, mx, 0.1, acc, stride, out, od, None, ws,
              wsb, 0, None)


def _prefill(q8=False, lay=None, bad="", q=P, qd=F16, B=1, Hq=16, start=P, mq=4, total=4, pos0=P, lens=P, bt=P, mb=4,
             window=10, sink=2, out=P, od=BF16, ws=P, wsb=BIG, sc=P, scb=BIG, scale=0.1):
    fn = L.lib().lstk_cuda_attn_prefill_window_q8 if q8 else L.lib().lstk_cuda_attn_prefill_window
    return fn(lay or _layout(), *_caches(q8, bad), q, qd, B, Hq, start, mq, total, pos0, lens, bt, mb, window, sink, scale,
              out, od, ws, wsb, *((sc, scb) if q8 else ()), None)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("call", [_window, _weights, _prefill])
def test_attention_refusals(call, q8):
    f = lambda **kw: call(q8=q8, **kw)  # noqa: E731
    assert f(lay=_layout(hd=64)) == UNSUP and "head_dim" in _lib.last_error()
    assert f(lay=_layout(bs=16)) == UNSUP
    assert f(lay=_layout(n_cells=33)) == ARG
    assert f(bad="k") == ARG and f(lens=None) == ARG and f(bt=None) == ARG and f(out=None) == ARG and f(q=None) == ARG
    assert f(qd=BF16) == UNSUP and f(od=F16) == UNSUP and f(od=7) == UNSUP
    assert f(B=-1) == ARG and f(Hq=12) == ARG and f(Hq=0) == ARG and f(mb=0) == ARG and f(mb=1 << 27) == ARG
    assert f(lay=_layout(hkv=1), Hq=16) == UNSUP
    assert f(q=P + 4) == ARG and f(out=P + 8) == ARG
    assert f(B=0) == _lib.LSTK_OK
    name = {_window: "attn_decode_window", _weights: "attn_decode_weights", _prefill: "attn_prefill_window"}[call]
    assert f(Hq=12) == ARG and ("lstk_cuda_" + name + ("_q8" if q8 else "")) in _lib.last_error()


@pytest.mark.parametrize("q8", [False, True])
def test_window_refusals(q8):
    for call in (_window, _prefill):
        for window, sink in ((0, 0), (-1, 4), (5, -1), (-2**31, 0)):
            assert call(q8=q8, window=window, sink=sink) == ARG and "window" in _lib.last_error()
    assert _window(q8=q8, ws=None) == ARG and _window(q8=q8, ws=P + 16) == ARG and _window(q8=q8, wsb=100) == CAP
    assert _window(q8=q8, B=5000) == CAP
    assert _prefill(q8=q8, qd=F32, wsb=100) == CAP and _prefill(q8=q8, qd=F32, ws=None) in (ARG, CAP)
    assert _prefill(q8=q8, lay=_layout(hkv=4), Hq=12) == UNSUP  # a group of 3 does not tile 128 rows
    size = L.lib().lstk_cuda_attn_prefill_window_workspace_size
    plain = L.lib().lstk_cuda_attn_prefill_workspace_size
    for bad in ((-1, 16, 8, 128, 4, 4, 4, F32, 10, 2), (1, 0, 8, 128, 4, 4, 4, F32, 10, 2), (1, 16, 8, 128, 4, 4, 4, F32, 0, 2),
                (1, 16, 8, 128, 4, 4, -4, F32, 10, 2)):
        assert size(*bad) == plain(*bad[:8])  # no split for what the call refuses
    assert size(1, 16, 8, 128, 4, 4, 4, F32, 10, 2) >= plain(1, 16, 8, 128, 4, 4, 4, F32)
    for scale in (0.0, -0.1, float("nan"), float("inf")):
        assert _prefill(q8=q8, scale=scale) == ARG and "scale" in _lib.last_error()
    assert _prefill(q8=q8, pos0=None) == ARG and _prefill(q8=q8, total=-1) == ARG
    if q8:
        assert _prefill(q8=True, sc=None) == ARG and _prefill(q8=True, scb=10) == CAP and _prefill(q8=True, sc=P + 16) == ARG


@pytest.mark.parametrize("q8", [False, True])
def test_weights_refusals(q8):
    f = lambda **kw: _weights(q8=q8, **kw)  # noqa: E731
    assert f(acc=None) == ARG and f(acc=P + 2) == ARG
    assert f(stride=127) == ARG and f(mx=100, stride=99) == ARG and "acc" in _lib.last_error()
    need = L.lib().lstk_cuda_attn_decode_weights_workspace_size(1, 16, 8, 128, 128)
    assert need > L.lib().lstk_cuda_attn_decode_workspace_size(1, 16, 8, 128) + 16 * 128 * 4
    assert f(wsb=need - 1) == CAP and f(ws=None) == ARG
    size = L.lib().lstk_cuda_attn_decode_weights_workspace_size
    assert size(-1, 16, 8, 128, 10) == 0 and size(1, 12, 8, 128, 10) == 0 and size(1, 16, 8, 128, -1) == 0
    # records past 32 bits: 4096 sequences of a million keys
    assert size(4096, 64, 8, 128, 1 << 20) > 4096 * (1 << 20) * 64 * 4


def _state(**kw):
    d = dict(acc=P, pos=P, held=P, shift=P, n_rows=2, row_cells=128)
    d.update(kw)
    return ctypes.byref(_lib.KvWeightsState(*d.values()))


def test_eviction_refusals():
    lib = L.lib()
    sel = lambda w=None, lens=P, budget=64, sink=4, recent=8, cap=64, n=P, s=P, d=P: lib.lstk_cuda_kv_evict_select(  # noqa: E731
        w or _state(), lens, budget, sink, recent, cap, n, s, d, None)
    assert sel(w=_state(acc=0)) == ARG and sel(w=_state(held=0)) == ARG and sel(w=_state(row_cells=0)) == ARG
    assert sel(w=_state(n_rows=-1)) == ARG and lib.lstk_cuda_kv_evict_select(None, P, 1, 0, 0, 64, P, P, P, None) == ARG
    assert sel(budget=0) == ARG and sel(sink=-1) == ARG and sel(recent=-1) == ARG and sel(sink=57) == ARG
    assert sel(budget=2**31 - 1, sink=2**31 - 1, recent=1) == ARG
    assert sel(cap=63) == CAP and sel(budget=100, cap=27) == CAP
    assert sel(lens=None) == ARG and sel(n=None) == ARG and sel(s=None) == ARG and sel(d=None) == ARG
    assert sel(w=_state(n_rows=0)) == _lib.LSTK_OK

    move = lambda lay=None, k=P, v=P, bt=P, rows=2, mb=4, n=P, s=P, d=P, cap=8: lib.lstk_cuda_kv_move(  # noqa: E731
        lay or _layout(), k, v, bt, rows, mb, n, s, d, cap, None)
    assert move(lay=_layout(hd=64)) == UNSUP and move(k=None) == ARG and move(v=None) == ARG and move(k=P + 8) == ARG
    assert move(bt=None) == ARG and move(n=None) == ARG and move(s=None) == ARG and move(rows=-1) == ARG
    assert move(mb=0) == ARG and move(mb=1 << 27) == ARG and move(cap=-1) == ARG
    assert move(rows=0) == _lib.LSTK_OK and move(cap=0, s=None, d=None) == _lib.LSTK_OK
    mq8 = lambda k=P, kd=P, v=P, vd=P, rows=2: lib.lstk_cuda_kv_move_q8(_layout(), k, kd, v, vd, P, rows, 4, P, P, P, 8, None)  # noqa: E731
    assert mq8(k=None) == ARG and mq8(vd=None) == ARG and mq8(v=P + 8) == ARG and mq8(kd=P + 4) == ARG
    assert mq8(rows=0) == _lib.LSTK_OK

    st = lambda slots=2, mb=4, bs=32: ctypes.byref(_lib.KvPages(P, P, P, P, P, slots, mb, bs))  # noqa: E731
    fin = lambda s=None, w=None, budget=64, cap=64, n=P, a=P, d=P: lib.lstk_cuda_kv_evict_finish(  # noqa: E731
        s or st(), w or _state(), budget, n, a, d, cap, None)
    assert fin(s=st(bs=16)) == UNSUP and fin(s=st(slots=3)) == ARG and fin(s=st(mb=5)) == ARG and fin(w=_state(pos=0)) == ARG
    assert fin(budget=0) == ARG and fin(cap=10) == ARG and fin(n=None) == ARG and fin(a=None) == ARG
    assert fin(s=st(mb=1 << 27)) == ARG


def test_finish_checks_its_moves():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    w = L.KvWeights(2, 4, device="cpu")
    for moves in (L.KvMoves(i32(3), i32(3, 64), i32(3, 64), 64), L.KvMoves(i32(2), i32(2, 64), i32(2, 63), 64),
                  L.KvMoves(i32(2).long(), i32(2, 64), i32(2, 64), 64), L.KvMoves(i32(2), i32(64, 2).t(), i32(2, 64), 64)):
        with pytest.raises(ValueError):
            w.finish(None, moves)


def test_python_checks():
    """The wrappers refuse shapes and types before any call (tensors on the CPU never reach the library)."""
    kc = torch.zeros(64, 2, 128, dtype=torch.float16)
    q = torch.zeros(2, 8, 128, dtype=torch.float16)
    bt, lens = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    acc = torch.zeros(2, 64)
    bad = [
        lambda: L.attn_decode_window(kc, kc[:32], q, bt, lens, 5),
        lambda: L.attn_decode_window(kc, kc, q[:, :, :64], bt, lens, 5),
        lambda: L.attn_decode_window(kc, kc, q.bfloat16(), bt, lens, 5),
        lambda: L.attn_decode_window(kc, kc, q, bt.long(), lens, 5),
        lambda: L.attn_decode_window(kc, kc, q, bt[:1], lens, 5),
        lambda: L.attn_decode_window(kc, kc, q, bt, lens[:1], 5),
        lambda: L.attn_decode_window(kc, kc, q, bt.t(), lens, 5),
        lambda: L.attn_decode_window(kc, kc, q, bt, lens, 5, out_dtype=torch.float16),
        lambda: L.attn_decode_window(kc, kc, q, bt, lens, 5, out=torch.zeros(2, 8, 64)),
        lambda: L.attn_decode_window(kc, kc, q, bt, lens, 5, lse_out=torch.zeros(2, 4)),
        lambda: L.attn_decode_weights(kc, kc, q, bt, lens, acc.half()),
        lambda: L.attn_decode_weights(kc, kc, q, bt, lens, acc[:1]),
        lambda: L.attn_decode_weights(kc, kc, q, bt, lens, acc[:, :60]),
        lambda: L.attn_decode_weights(kc, kc, q, bt, lens, acc.t().contiguous().t()),
        lambda: L.attn_decode_weights(kc, kc, q, bt, lens, torch.zeros(64).expand(2, 64)),
        lambda: L.attn_prefill_window(kc, kc, q, lens, lens, lens, bt, 1, 5),
        lambda: L.attn_prefill_window(kc, kc, q.transpose(0, 1), torch.zeros(3, dtype=torch.int32), lens, lens, bt, 1, 5),
        lambda: L.attn_prefill_window(kc, kc, q, torch.zeros(3, dtype=torch.int32), lens, lens, bt, 1, 5,
                                      workspace=torch.zeros(1, dtype=torch.uint8).expand(1 << 20)),
        lambda: L.Q8Cache.from_planes(torch.zeros(33, 2, 128, dtype=torch.int8), torch.zeros(33, 2, 4).half()),
        lambda: L.Q8Cache.from_planes(torch.zeros(32, 2, 128, dtype=torch.int8), torch.zeros(32, 2, 3).half()),
        lambda: L.KvWeights.from_tensors(acc, torch.zeros(2, 63, dtype=torch.int32), lens, lens),
        lambda: L.KvWeights.from_tensors(acc.double(), torch.zeros(2, 64, dtype=torch.int32), lens, lens),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
