"""Calls of paged_attention whose parts a second launch joins: their parts are the call's own, so host threads
that share a stream do not see each other's."""
import ctypes
import threading

import pytest
import torch

from test_paged_attention_gpu import check, make

pytestmark = pytest.mark.gpu


def two_calls(gpu):
    """Arguments of two calls that a second kernel joins, of different shapes and cuts."""
    from powershard_amd import _native
    calls = [make([30000], 8, 1, 128, 16, "int8", torch.bfloat16, gpu, seed=1),
             make([5000, 1200, 6000], 16, 1, 256, 48, "fp8", torch.float16, gpu, seed=2)]
    for q, k, v, table, *_ in calls:
        code = _native.CODES_I8 if k.dtype is torch.int8 else _native.CODES_E4M3
        assert _native.lib().psq_paged_attention_own_workspace(code, len(q), q.shape[1], 1, q.shape[2], table.shape[1] * k.shape[2]) == 1
    return calls


@pytest.mark.parametrize("direct", [True, False])
def test_parts_are_not_in_the_streams_workspace(gpu, monkeypatch, direct):
    """The workspace that a call of two launches passes (recorded in place of the library's entry point)."""
    from powershard_amd import _native, ops
    entry = _native.lib().psq_paged_attention
    args = two_calls(gpu)[0]
    device, stream = gpu.index or 0, torch.cuda.current_stream(gpu).cuda_stream or None
    ops._workspace(torch.device("cuda", device), stream, 1 << 25)   # the stream has one that is large enough
    seen = []
    kind = ctypes.CFUNCTYPE(entry.restype, *entry.argtypes)
    recorder = kind(lambda *a: seen.append((a[-3], a[-2])) or 0)
    module = _native.direct()
    if direct:
        names = {n: ctypes.cast(getattr(_native.lib(), n), ctypes.c_void_p).value for n in _native.DIRECT_CALLS}
        module.bind(dict(names, psq_paged_attention=ctypes.cast(recorder, ctypes.c_void_p).value))
    else:
        monkeypatch.setattr(_native, "_direct", False)
        monkeypatch.setattr(_native.lib(), "psq_paged_attention", recorder)
    try:
        ops.paged_attention(*args)
    finally:
        if direct:
            module.bind(names)
    (address, size), = seen
    need = _native.lib().psq_paged_attention_workspace_bytes(_native.CODES_I8, 1, 8, 1, 128, args[3].shape[1] * 16)
    assert size >= need > 0 and address % 256 == 0
    for held in ops._workspaces.values():
        assert address + size <= held.data_ptr() or address >= held.data_ptr() + held.numel()


def test_two_host_threads_on_one_stream(gpu):
    """Each thread's results have the bits of single calls, whatever the other enqueues in between."""
    from powershard_amd import ops
    calls = two_calls(gpu)
    want = [ops.paged_attention(*args) for args in calls]
    for got, args in zip(want, calls):
        check(got, args)
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(2)

    def work(args, first):
        start.wait()
        for i in range(400):
            if not torch.equal(ops.paged_attention(*args), first):
                wrong.append(i)
    threads = [threading.Thread(target=work, args=pair) for pair in zip(calls, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_no_expectation_past_the_table(gpu):
    """max_len beyond what the table holds plans as the table's length does: memory and plan agree."""
    from powershard_amd import ops
    for args in two_calls(gpu):
        assert torch.equal(ops.paged_attention(*args, max_len=1 << 40), ops.paged_attention(*args))
