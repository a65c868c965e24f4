"""Decode with accumulated weights after a wait that ran out: acc is updated in place, so a call that
reports LSTK_ERR_TIMEOUT leaves it as it was and can be repeated."""
import pytest
import torch

import localstack_b200 as L
from localstack_b200 import _lib
from tests.bounded_ref import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("lens,own_ws", [([4000, 33, 1, 700], True), ([4000, 33, 1, 700], False), ([40], True),
                                         ([0, 20000], True), (list(range(20, 900, 40)), True)])
def test_a_timeout_leaves_acc_and_the_call_can_be_repeated(lens, own_ws, q8):
    """The loaders are gated on a flag that nothing sets, with a limit of 2 ms (a host-visible status, no
    fault), over what earlier calls left in the workspace: scores and NaN."""
    Hq, Hkv = 16, 4
    b = Batch(lens, Hq, Hkv, seed=len(lens), q8=q8)
    acc = torch.rand((len(lens), b.bt.shape[1] * 32), generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    before = acc.clone()
    ws = L.WeightsWorkspace(len(lens), Hq, Hkv, acc.shape[1]) if own_ws else None
    fn = L.attn_decode_weights_q8 if q8 else L.attn_decode_weights
    call = lambda a: fn(*b.cache, b.q, b.bt, b.lens_t, a, workspace=ws)  # noqa: E731
    want = before.clone()
    out = call(want)
    L.check_status()
    assert not torch.equal(want, before)
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    for fill in (None, 0xff, 0):
        if own_ws and fill is not None:
            ws.buf.fill_(fill)
        _lib.check(L.lib().lstk_cuda_set_wait_policy(2_000_000, flag.data_ptr()))
        try:
            call(acc)
            with pytest.raises(L.LstkError) as e:
                L.check_status()
        finally:
            _lib.check(L.lib().lstk_cuda_set_wait_policy(0, None))
        assert e.value.code == _lib.LSTK_ERR_TIMEOUT
        assert torch.equal(acc, before)
    assert torch.equal(call(acc), out) and torch.equal(acc, want)
    L.check_status()
