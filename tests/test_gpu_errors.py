"""A call that fails in the CUDA runtime reports it once: the next, valid call is not blamed for it."""
import ctypes

import pytest
import torch

import localstack_b200 as L
from localstack_b200 import _lib
from tests.bounded_ref import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("op", ["decode", "window", "weights", "prefill"])
def test_an_error_is_reported_once(op):
    b = Batch([300], 16, 8, seed=1, q_dtype=torch.float32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    acc = torch.zeros(1, b.bt.shape[1] * 32, device="cuda")
    calls = dict(decode=lambda: L.attn_decode(*b.cache, b.q, b.bt, b.lens_t),
                 window=lambda: L.attn_decode_window(*b.cache, b.q, b.bt, b.lens_t, 99, 4),
                 weights=lambda: L.attn_decode_weights(*b.cache, b.q, b.bt, b.lens_t, acc),
                 prefill=lambda: L.attn_prefill(*b.cache, b.q, i32([0, 1]), i32([299]), b.lens_t, b.bt, 1))
    want = calls[op]()
    box, handle = ctypes.c_void_p(), (ctypes.c_char * 64)()
    rc = L.lib().lstk_cuda_mailbox_alloc(1 << 50, ctypes.byref(box), handle)  # more than any GPU has
    assert rc == _lib.LSTK_ERR_CUDA and "cudaMalloc" in _lib.last_error() and not box.value
    assert torch.equal(calls[op](), want)
    L.check_status()
