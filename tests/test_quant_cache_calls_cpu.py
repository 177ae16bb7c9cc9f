"""How the quantised cache's Python entries call the library, without a GPU: fake entries stand in for the C functions."""
import threading
import time

import pytest
import torch

from utmist_bigger_bird_b200 import _lib, quant_cache


@pytest.fixture
def calls(monkeypatch):
    """_run on a fake entry, as if no graph were captured; every call's (workspace, its size, tickets, their number)."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(quant_cache, "_scratch", {})
    seen = []

    def call(need=1000, tickets=16, during=None):
        a = _lib.QkvAttnArgs()

        def run(ref, ws, nbytes, stream):
            if nbytes < need:
                return _lib.BB_ERR_WORKSPACE
            seen.append((ws, nbytes, a.tickets, a.n_tickets))
            if during:
                during(ws, a.tickets)
            return 0

        def size_of(ref, size):
            size._obj.value = need
            return 0

        quant_cache._run("call", run, size_of, a, torch.device("cpu"), 0, tickets)

    call.seen = seen
    return call


def test_threads_on_one_stream_do_not_share_a_workspace_in_a_call(calls):
    """A call enqueues several launches that hand each other results in the workspace: no second call may use the same
    buffers until the first has enqueued its last."""
    busy, shared = set(), []

    def during(ws, tickets):
        shared.extend(x for x in (ws, tickets) if x in busy)
        busy.update((ws, tickets))
        time.sleep(0.02)
        busy.difference_update((ws, tickets))

    calls()  # the stream's buffers exist
    threads = [threading.Thread(target=calls, kwargs=dict(during=during)) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(calls.seen) == 5 and not shared


@pytest.fixture
def on_gpu_0(monkeypatch):
    """GPU 0 is current as far as the wrappers can tell; the GPU that is current, as a list of one."""
    current = [0]

    class Enter:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *exc):
            current[0] = self.before

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Enter)
    return current


@pytest.mark.parametrize("index", [0, 1])
def test_attention_calls_run_with_the_cache_s_gpu_current(on_gpu_0, monkeypatch, index):
    at = []

    def take(device, *args):
        at.append(on_gpu_0[0])
        return torch.zeros(8, dtype=torch.int32), torch.zeros(8, dtype=torch.uint8), threading.Lock()

    def run(*args):
        at.append(on_gpu_0[0])
        return 0

    monkeypatch.setattr(quant_cache, "_take_scratch", take)
    quant_cache._run("call", run, None, _lib.QkvAttnArgs(), torch.device("cuda", index), 0, 4)
    assert at == [index, index] and on_gpu_0 == [0]


@pytest.mark.parametrize("index", [0, 1])
def test_write_and_read_run_with_the_cache_s_gpu_current(on_gpu_0, monkeypatch, index):
    kv = quant_cache.QuantKV(2, 10, 64, device="cpu")
    at = []

    def stop(*args, **kw):
        at.append(on_gpu_0[0])
        raise RuntimeError("no further")

    class Rows:  # as far as write looks before it calls anything
        device, dtype, shape = torch.device("cuda", index), torch.bfloat16, (2, 3, 64)

    kv.device = torch.device("cuda", index)
    monkeypatch.setattr(quant_cache, "_rows", stop)
    monkeypatch.setattr(torch, "empty_strided", stop)
    for call in (lambda: kv.write(Rows(), Rows(), 0), lambda: kv.read()):
        with pytest.raises(RuntimeError, match="no further"):
            call()
    assert at == [index, index] and on_gpu_0 == [0]


def test_the_number_of_query_rows_is_bounded_by_32_bits_only():
    """Follow-up prompts: 32 heads x 4096 tokens and more are planned; the workspace holds no partial results where the
    query rows fill the GPU without cutting the keys."""
    import ctypes as C

    from test_quant_cache_cpu import BUF, attn
    L, size = _lib.lib(), C.c_size_t(0)
    big = dict(k_codes_h=64 * 2 ** 21, k_meta_h=4 * 2 ** 21, v_codes_h=64 * 2 ** 21, v_meta_h=4 * 2 ** 21, cap=2 ** 21)
    for t in (2047, 2048, 4096, 131072, 2 ** 25):
        a = attn(big, n=2 ** 21, t=t, window=2 ** 21, front=0)
        assert L.bb_qkv_decode_workspace_size(C.byref(a), C.byref(size)) == 0, t
        assert 0 < size.value <= 1 << 20, (t, size.value)
    a = attn(big, n=2 ** 21, t=2 ** 25 + 1, window=2 ** 21)
    assert L.bb_qkv_decode_workspace_size(C.byref(a), C.byref(size)) == 2 and "tokens" in L.bb_last_error().decode()
    a = attn(big, n=2 ** 21, t=2 ** 25, window=2 ** 21, splits=1000)   # no more CTAs than a grid has
    assert L.bb_qkv_decode_workspace_size(C.byref(a), C.byref(size)) == 0
    assert a.cache.k_codes == BUF


def test_kept_buffers_stay_whatever_the_calls_need(calls):
    """Calls of other sizes in between do not replace a stream's buffers, and a call too large for them gets its own."""
    calls()
    first = calls.seen[-1]
    for kw in (dict(need=100 << 20), dict(tickets=2000), dict(need=100 << 20), dict(tickets=70000, need=50 << 20)):
        calls(**kw)
        ws, nbytes, tickets, n_tickets = calls.seen[-1]
        assert nbytes >= kw.get("need", 0) and 0 < n_tickets <= kw.get("tickets", 16)
        calls()
        assert calls.seen[-1] == first
    assert len(quant_cache._scratch) == 1
    kept = sum(x.numel() * x.element_size() for s in quant_cache._scratch.values() for x in s if isinstance(x, torch.Tensor))
    assert kept <= 16 << 20


def test_a_captured_call_fills_its_counters_once(calls, monkeypatch):
    """Every fill under a capture is a node that each replay pays for. A captured call uses nothing of the kept buffers."""
    calls()
    filled, zeros = [], torch.zeros
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(torch, "zeros", lambda *a, **kw: filled.append(zeros(*a, **kw)) or filled[-1])
    for need in (1000, 100 << 20):
        calls(need=need)
        assert len(filled) == 1 and calls.seen[-1][2] == filled.pop().data_ptr()
        assert calls.seen[-1][0] != calls.seen[0][0] and calls.seen[-1][2] != calls.seen[0][2]
