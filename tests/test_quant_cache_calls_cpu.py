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
