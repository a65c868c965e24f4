"""The bounded-cache wrappers and Python threads: a call that waits for room in the stream's queue lets other
threads run, and calls from several threads at once are right."""
import threading
import time

import pytest
import torch

import localstack_b200 as L
from localstack_b200 import _lib
from tests.bounded_ref import Batch

pytestmark = pytest.mark.gpu


def test_a_call_that_waits_for_the_queue_lets_other_threads_run():
    """The first call's loaders wait for a flag in pinned host memory (2 s at most, a status and no fault); calls
    are issued behind it until the queue is full and one of them waits. Another thread then sets the flag.
    Were the interpreter locked meanwhile, that would come only after the wait had run out."""
    b = Batch([300], 16, 8, seed=1)
    flag, ws = torch.zeros(1, dtype=torch.int32).pin_memory(), L.DecodeWorkspace(1, 16, 8)
    opened = flag.numpy()
    out = torch.empty(1, 16, 128, device="cuda")
    call = lambda: L.attn_decode_window(*b.cache, b.q, b.bt, b.lens_t, 99, 4, out=out, workspace=ws)  # noqa: E731
    want = call().clone()
    L.check_status()
    set_at, longest = [], 0.0

    def opener():
        time.sleep(0.3)
        opened[0] = 1
        set_at.append(time.perf_counter())

    t = threading.Thread(target=opener)
    begin = time.perf_counter()
    t.start()
    _lib.check(L.lib().lstk_cuda_set_wait_policy(2_000_000_000, flag.data_ptr()))
    try:
        call()
    finally:
        _lib.check(L.lib().lstk_cuda_set_wait_policy(0, None))
    for _ in range(3000):  # two launches each: more than a queue holds
        at = time.perf_counter()
        call()
        longest = max(longest, time.perf_counter() - at)
        if set_at:
            break
    t.join()
    torch.cuda.synchronize()
    L.check_status()  # no wait ran out
    assert torch.equal(out, want)
    assert longest > 0.05, "the queue never filled, so nothing was tested"
    assert set_at[0] - begin < 1.0


@pytest.mark.parametrize("q8", [False, True])
def test_calls_from_several_threads(q8):
    """Each thread on a stream of its own, with its own sequences: the results of the same calls made alone."""
    sfx = "_q8" if q8 else ""
    batches = [Batch([700 + 31 * i, 5, 64 * i + 1], 16, 4, seed=i, q8=q8) for i in range(4)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    start = i32([0, 1, 2, 3])

    def calls(b, acc, stream):
        w = L.KvWeights.from_tensors(acc, torch.zeros_like(acc, dtype=torch.int32), i32([0] * 3), i32([0] * 3))
        o = [getattr(L, "attn_decode_window" + sfx)(*b.cache, b.q, b.bt, b.lens_t, 200, 4, stream=stream),
             getattr(L, "attn_decode_weights" + sfx)(*b.cache, b.q, b.bt, b.lens_t, acc, stream=stream),
             getattr(L, "attn_prefill_window" + sfx)(*b.cache, b.q, start, b.lens_t - 1, b.lens_t, b.bt, 1, 200, 4, stream=stream)]
        m = w.select(b.lens_t, 100, 4, 10, stream=stream)
        return o + [acc, m.n, m.src, m.dst]

    accs = [torch.zeros(3, b.bt.shape[1] * 32, device="cuda") for b in batches]
    want = [calls(b, a, None) for b, a in zip(batches, accs)]
    torch.cuda.synchronize()
    L.check_status()
    got, errors = [None] * 4, []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(25):
                    acc = torch.zeros_like(accs[i])
                    got[i] = calls(batches[i], acc, None)
                s.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    L.check_status()
    assert not errors, errors
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
