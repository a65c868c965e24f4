"""Decode attention that accumulates the keys' attention weights, against f64 (bounds:
tests/bounded_ref.py; the accumulated sums add 2^-24 per f32 addition)."""
import numpy as np
import pytest
import torch

import localstack_b200 as L
from localstack_b200 import _lib
from tests.bounded_ref import Batch, close

pytestmark = pytest.mark.gpu


def _run(b, acc, **kw):
    fn = L.attn_decode_weights_q8 if b.q8 else L.attn_decode_weights
    out, lse = fn(*b.cache, b.q, b.bt, b.lens_t, acc, want_lse=True, **kw)
    L.check_status()
    return out, lse


def _acc(b, seed=0, fill=None, pad=0):
    width = b.bt.shape[1] * 32 + pad
    if fill is not None:
        return torch.full((len(b.lens), width), fill, device="cuda")
    return torch.rand((len(b.lens), width), generator=torch.Generator("cuda").manual_seed(seed), device="cuda")


def _check(b, out, lse, acc, before, steps=1):
    bf16 = out.dtype == torch.bfloat16
    out, lse, acc = out.float().cpu().numpy(), lse.cpu().numpy(), acc.cpu().numpy().astype(np.float64)
    before = before.cpu().numpy().astype(np.float64)
    for i, n in enumerate(b.lens):
        o, l, w, t_o, t_l, t_w = b.decode_ref(i)
        close(out[i:i + 1], o, t_o, bf16, f"out of length {n}")
        close(lse[i:i + 1], l, t_l, False, f"lse of length {n}")
        want = before[i, :n] + steps * w
        # Hq f32 additions per key and step, and one per step onto the accumulated value
        close(acc[i, :n], want, steps * (t_w + b.Hq * 2.0 ** -24 * w + 2.0 ** -24 * want), False, f"weights of length {n}")
        assert np.array_equal(acc[i, n:], before[i, n:])  # entries behind the sequence stay


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("Hq,Hkv", [(32, 4), (16, 8), (28, 4), (12, 2), (48, 12), (20, 10)])
def test_weights(Hq, Hkv, q8):
    b = Batch([0, 1, 31, 32, 33, 257, 1000, 0], Hq, Hkv, seed=Hq + Hkv, q8=q8)
    acc = _acc(b)
    before = acc.clone()
    out, lse = _run(b, acc)
    _check(b, out, lse, acc, before)


@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (4, 4), (5, 5)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_dtype", [torch.float16, torch.float32])
def test_types(Hq, Hkv, out_dtype, q_dtype):
    b = Batch([100, 3, 640], Hq, Hkv, seed=Hq, q_dtype=q_dtype)
    acc = _acc(b, fill=0.0)
    before = acc.clone()
    out, lse = _run(b, acc, out_dtype=out_dtype)
    assert out.dtype == out_dtype
    _check(b, out, lse, acc, before)
    # every head's weights sum to 1
    assert np.allclose(acc.sum(1).cpu().numpy(), Hq, rtol=1e-4)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("lens", [[4000], [20000], [5000, 3, 17, 9000], list(range(1, 2000, 37))])
@pytest.mark.parametrize("n_ctas", [0, 3, 300])
def test_splits(lens, n_ctas, q8):
    b = Batch(lens, 32, 4, seed=len(lens) + n_ctas, q8=q8)
    acc = _acc(b, fill=0.0)
    before = acc.clone()
    out, lse = _run(b, acc, n_ctas=n_ctas, out_dtype=torch.bfloat16)
    _check(b, out, lse, acc, before)


def test_matches_attn_decode_and_repeats_its_bits():
    b = Batch([0, 700, 33, 4097], 32, 4, seed=4)
    ref, ref_lse = L.attn_decode(*b.cache, b.q, b.bt, b.lens_t, want_lse=True)
    accs = []
    for _ in range(3):
        acc = _acc(b)
        out, lse = _run(b, acc)
        assert torch.equal(out, ref) and torch.equal(lse, ref_lse)
        accs.append(acc)
    assert torch.equal(accs[0], accs[1]) and torch.equal(accs[0], accs[2])


def test_strided_rows_several_steps_and_no_lse():
    b = Batch([40, 500, 0, 64], 16, 8, seed=5)
    whole = _acc(b, pad=50)
    acc = whole[:, 3:-5]  # rows at a stride, starting off a 16-byte boundary
    before, edges = acc.clone(), whole.clone()
    for _ in range(3):
        out = L.attn_decode_weights(*b.cache, b.q, b.bt, b.lens_t, acc)
    L.check_status()
    _, lse = _run(b, _acc(b))
    _check(b, out, lse, acc, before, steps=3)
    assert torch.equal(whole[:, :3], edges[:, :3]) and torch.equal(whole[:, -5:], edges[:, -5:])


@pytest.mark.parametrize("q8", [False, True])
def test_hidden_cells_do_not_matter(q8):
    b = Batch([45, 500, 64], 16, 8, seed=6, q8=q8)
    acc, again = _acc(b), _acc(b)
    out, lse = _run(b, acc)
    b.poison([np.arange(n) for n in b.lens])
    out2, lse2 = _run(b, again)
    assert torch.equal(out, out2) and torch.equal(lse, lse2) and torch.equal(acc, again)


def test_max_seq_len_bounds_what_is_attended_to():
    """The records hold max_seq_len keys: a longer sequence reports it and stops there."""
    b = Batch([300, 100], 32, 4, seed=7)
    acc = _acc(b)
    before = acc.clone()
    out = L.attn_decode_weights(*b.cache, b.q, b.bt, b.lens_t, acc, max_seq_len=130)
    with pytest.raises(L.LstkError) as e:
        L.check_status()
    assert e.value.code == _lib.LSTK_ERR_DEVICE_INDEX
    lse = torch.zeros(2, 32)
    b.lens = [130, 100]
    for i in range(2):
        lse[i] = torch.from_numpy(b.decode_ref(i)[1][0])
    _check(b, out, lse, acc, before)


def test_a_bad_page_has_no_weight():
    b = Batch([100], 32, 4, seed=8)
    b.bt[0, 1] = -3
    ws = L.WeightsWorkspace(1, 32, 4, b.bt.shape[1] * 32)
    ws.buf.fill_(0x7f)  # whatever an earlier call left there
    acc = _acc(b)
    before = acc.clone()
    out = L.attn_decode_weights(*b.cache, b.q, b.bt, b.lens_t, acc, workspace=ws)
    with pytest.raises(L.LstkError) as e:
        L.check_status()
    assert e.value.code == _lib.LSTK_ERR_DEVICE_INDEX
    assert torch.isfinite(out).all() and torch.equal(acc[0, 32:64], before[0, 32:64])
    assert (acc[0, :32] > before[0, :32]).all() and np.isclose((acc - before).sum().item(), 32, rtol=1e-3)


def test_graph_on_another_stream():
    b = Batch([400, 90, 65], 32, 4, seed=9)
    acc = _acc(b, fill=0.0)
    out, lse = torch.empty_like(b.q, dtype=torch.bfloat16), torch.empty(3, 32, device="cuda")
    ws = L.WeightsWorkspace(3, 32, 4, b.bt.shape[1] * 32)
    call = lambda: L.attn_decode_weights(*b.cache, b.q, b.bt, b.lens_t, acc, out=out, lse_out=lse, want_lse=True,  # noqa: E731
                                         workspace=ws)
    call()
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        call()
    for lens in ([400, 90, 65], [33, 0, 1]):
        b.lens = lens
        b.lens_t.copy_(torch.tensor(lens, dtype=torch.int32))
        acc.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
            g.replay()
        torch.cuda.synchronize()
        L.check_status()
        _check(b, out, lse, acc, torch.zeros_like(acc), steps=2)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("lens", [[20, 300], [600, 300], [5000, 300], list(range(20, 900, 40))])
def test_a_nan_key_makes_its_rows_nan(lens, q8):
    b = Batch(lens, 16, 4, seed=1, q8=q8)
    for i in range(len(lens) - 1):
        (b.cache[0].d if q8 else b.cache[0])[b.cells(i)[lens[i] - 5], 2] = float("nan")
    acc = _acc(b)
    before = acc.clone()
    out, lse = _run(b, acc)
    group = slice(8, 12)
    assert out[:-1, group].isnan().all() and lse[:-1, group].isnan().all()
    for i, n in enumerate(lens[:-1]):
        assert acc[i, :n].isnan().all() and torch.equal(acc[i, n:], before[i, n:])
    out[:-1, group] = 0
    assert not out.isnan().any() and not acc[-1].isnan().any()


@pytest.mark.parametrize("Hq,Hkv", [(16, 8), (32, 4), (12, 12)])
@pytest.mark.parametrize("q8", [False, True])
def test_one_sequence_in_a_long_table(Hq, Hkv, q8):
    """Fewer pages than CTAs: some CTAs have none, and what earlier calls left in the workspace stays out."""
    ws = L.WeightsWorkspace(1, Hq, Hkv, 12800 + 4800)
    ws.buf.fill_(0xff)  # NaN
    for n in (1, 32, 33, 64, 65, 100, 513, 1000, 2047, 2400, 4700, 0, 40):
        b = Batch([n], Hq, Hkv, seed=n, q8=q8)
        b.bt = torch.cat([b.bt, b.bt[:, :1].expand(1, 400)], 1)
        acc = _acc(b)
        before = acc.clone()
        out, lse = _run(b, acc, workspace=ws)
        _check(b, out, lse, acc, before)
