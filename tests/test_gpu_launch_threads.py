"""GPU: calls of the C ABI from two host threads at once, of sizes that want different amounts of shared memory of the
same kernel: every call launches."""
import ctypes
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _together(calls, times):
    """The calls in a thread each, `times` times; their statuses other than 0."""
    bad = [[] for _ in calls]
    start = threading.Barrier(len(calls))

    def work(k):
        start.wait()
        for _ in range(times):
            status = calls[k]()
            if status:
                bad[k].append(status)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return bad


def test_state_rows():
    from burn_gdn2 import LIB, _lib

    def call(rows):
        pool = torch.zeros(rows, 16, device="cuda")
        index = torch.arange(rows, dtype=torch.int32, device="cuda").roll(1)
        t = (_lib.StateRows * 1)(_lib.StateRows(pool.data_ptr(), pool.data_ptr(), 64))
        stream = torch.cuda.Stream()
        keep = (pool, index, stream)
        return lambda: LIB.gdn2_move_state_rows(t, 1, index.data_ptr(), rows, rows, stream.cuda_stream) if keep else 1

    calls = [call(8), call(4096)]
    torch.cuda.synchronize()
    assert _together(calls, 4000) == [[], []]


def test_wide_group_norm():
    from burn_gdn2 import LIB, _lib

    def call(width):
        x, dy, dx = (torch.ones(1, width, device="cuda") for _ in range(3))
        w, b, dw, db = (torch.ones(width, device="cuda") for _ in range(4))
        p = lambda t: t.data_ptr()
        a = _lib.GroupNormArgs(1, 1, width, 0, 1, 0, 1e-5, p(x), width, None, 0, p(w), p(b))
        bwd = _lib.GroupNormBwdArgs(a, p(dy), width, p(dx), None, p(dw), p(db))
        need = LIB.gdn2_group_norm_gate_bwd_workspace_bytes(ctypes.byref(bwd))
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        stream = torch.cuda.Stream()
        keep = (x, dy, dx, w, b, dw, db, ws, stream)
        return lambda: LIB.gdn2_group_norm_gate_bwd(ctypes.byref(bwd), p(ws), need, stream.cuda_stream) if keep else 1

    calls = [call(4100), call(12288)]
    torch.cuda.synchronize()
    assert _together(calls, 4000) == [[], []]
