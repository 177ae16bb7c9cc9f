"""The quantised routing's bounded wait, on the GPU, without a GPU fault.

The CTAs of a KV head wait for each other's statistics until as many as there are have arrived, by a counter that starts at
zero. A counter that starts far below zero stands for CTAs that never arrive: the wait runs out (after a limit that
``bb_set_wait_limit_ns`` shortens), code 48 is recorded, the probabilities of that KV head are NaN, and the counters are
zero afterwards, so that the next call is right."""
import ctypes as C

import pytest
import torch

from test_gpu_quant_cache import filled, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


def fault():
    from utmist_bigger_bird_b200 import _lib
    code = C.c_int(-1)
    _lib.check(_lib.lib().bb_device_fault(C.byref(code)), "device_fault")
    return code.value


@pytest.mark.parametrize("g,bits,d", [(4, 4, 128), (8, 8, 96)])
def test_a_wait_that_runs_out_is_reported_and_leaves_the_next_call_right(g, bits, d):
    from utmist_bigger_bird_b200 import _lib, quant_cache, quant_pooled_probs, quant_route
    L = _lib.lib()
    hk, cap, n = 2, 6000, 5990
    kv, *_ = filled(hk, cap, d, bits, 32)
    q = rand((hk * g, 1, d), 40)[:, 0]
    kw = dict(front=5, window=77, scale=d ** -0.5, n=n)
    want, routes = quant_pooled_probs(q, kv, **kw), quant_route(q, kv, 32, **kw)
    torch.cuda.synchronize()
    assert fault() == 0
    tickets, *_ = quant_cache._scratch[kv.device.index, torch.cuda.current_stream().cuda_stream]
    assert not tickets.any()
    _lib.check(L.bb_set_wait_limit_ns(20_000_000), "set_wait_limit_ns")
    try:
        tickets[2] = -1000                                  # arrivals of KV head 1
        late = quant_pooled_probs(q, kv, **kw)
        torch.cuda.synchronize()
    finally:
        _lib.check(L.bb_set_wait_limit_ns(2_000_000_000), "set_wait_limit_ns")
    assert fault() == 48 and fault() == 0
    assert not tickets.any()
    assert torch.equal(late[0], want[0])
    live = want[1] != -1
    assert torch.isnan(late[1, live]).all() and (late[1, ~live] == -1).all()
    for _ in range(3):
        assert torch.equal(quant_pooled_probs(q, kv, **kw), want) and torch.equal(quant_route(q, kv, 32, **kw), routes)
    assert fault() == 0
