"""ops._workspace: the buffer that the calls of a stream share (on the CPU, with plain host memory)."""
import sys
import threading

import pytest
import torch

from powershard_amd import ops

CPU = torch.device("cpu")


@pytest.fixture
def empty(monkeypatch):
    monkeypatch.setattr(ops, "_workspaces", {})
    monkeypatch.setattr(ops, "_retired_workspaces", [])
    state = {"capturing": False}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    return state


def test_grows_and_keeps_the_old_one(empty):
    a, n = ops._workspace(CPU, 1, 100)
    assert n == a.numel() == ops._WS_MIN_BYTES and not a.any()
    assert ops._workspace(CPU, 1, 200)[0] is a and ops._workspace(CPU, 2, 1)[0] is not a
    b, n = ops._workspace(CPU, 1, ops._WS_MIN_BYTES + 1)
    assert n == 2 * ops._WS_MIN_BYTES and ops._retired_workspaces == [a] and ops._workspace(CPU, 1, 1)[0] is b
    assert ops._workspace(CPU, 1, 0) == (None, 0)


def test_none_is_made_or_replaced_during_a_capture(empty):
    """Its zeros would be recorded in the graph and only its replays would write them."""
    empty["capturing"] = True
    assert ops._workspace(CPU, 1, 100) == (None, 0) and not ops._workspaces
    empty["capturing"] = False
    held, n = ops._workspace(CPU, 1, 100)
    empty["capturing"] = True
    assert ops._workspace(CPU, 1, n)[0] is held
    assert ops._workspace(CPU, 1, n + 1) == (None, 0)
    assert list(ops._workspaces.values()) == [held] and not ops._retired_workspaces


def test_host_threads(empty, monkeypatch):
    """Threads that meet in a new stream's first call, or in other streams' ones: one workspace per stream, and no
    thread trips over another's entry."""
    monkeypatch.setattr(ops, "_MAX_WS_STREAMS", 10000)
    monkeypatch.setattr(ops, "_WS_MIN_BYTES", 16)
    old = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        got, errors, start = [[] for _ in range(4)], [], threading.Barrier(4)

        def work(mine):
            start.wait()
            try:
                for stream in range(500):
                    mine.append(ops._workspace(CPU, stream, 8)[0])
            except RuntimeError as error:
                errors.append(error)
        threads = [threading.Thread(target=work, args=(mine,)) for mine in got]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(old)
    assert not errors
    for same in zip(*got):
        assert all(ws is same[0] for ws in same)
