"""Calls of several host threads on one stream, which share its scratch: a call's launches stay together."""
import ctypes
import threading

import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import _lib

pytestmark = pytest.mark.gpu
THREADS, CALLS = 4, 1000


def ptr(t):
    return ctypes.c_void_p(t.data_ptr())


def scratch(nbytes):
    return torch.zeros(nbytes, dtype=torch.uint8, device="cuda")


def run_threads(call, shape):
    """call(thread, where the result goes), straight into the library, which Python calls without its own lock: THREADS threads, CALLS
    calls each, nothing between two calls.  Every result is compared with the thread's first one, which is computed alone."""
    out = torch.empty((THREADS, CALLS + 1) + shape, dtype=torch.bfloat16, device="cuda")
    jobs = [[call(i, out[i, c]) for c in range(CALLS + 1)] for i in range(THREADS)]
    for i in range(THREADS):
        _lib.check(jobs[i][0]())
    torch.cuda.synchronize()
    codes, gate = [0] * THREADS, threading.Barrier(THREADS)

    def work(i):
        gate.wait()
        for job in jobs[i][1:]:
            codes[i] |= job()

    ts = [threading.Thread(target=work, args=(i,)) for i in range(THREADS)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    torch.cuda.synchronize()
    assert codes == [0] * THREADS
    assert torch.isfinite(out).all()
    assert not any(torch.equal(out[0, 0], out[i, 0]) for i in range(1, THREADS))
    same = (out == out[:, :1]).flatten(2).all(2).sum(1).tolist()
    assert same == [CALLS + 1] * THREADS


def bound(f, *a):
    """f with its arguments converted once."""
    a = [t(v) if not isinstance(v, t) else v for t, v in zip(f.argtypes, a)]
    return lambda: f(*a)


@pytest.mark.parametrize("mode", (_lib.MXFP4, _lib.NVFP4))
def test_qqmm(mode):
    lib, T, N, K = _lib.load(), 16, 256, 1024
    w, s = mb.quantize(torch.randn(N, K, device="cuda").bfloat16(), mode=("mxfp4", "nvfp4")[mode])
    xs = torch.randn(THREADS, T, K, device="cuda").bfloat16()
    ws = scratch(lib.b200q_grouped_qqmm_workspace_bytes(T, 1, N, K, mode))
    run_threads(lambda i, y: bound(lib.b200q_grouped_qqmm, ptr(xs[i]), ptr(w), ptr(s), None, 0, ptr(y), _lib.BF16, T, 1, N, K, mode, None, None, 0,
                                   ptr(ws), ws.numel(), None), (T, N))


def test_grouped_mm_of_rows_off_16_byte_boundaries():
    lib, T, E, N, K = _lib.load(), 16, 2, 96, 255
    w, n = torch.randn(E, N, K, device="cuda").bfloat16(), torch.tensor([9, 7], device="cuda")
    xs = torch.randn(THREADS, 4096, device="cuda").bfloat16()   # (each on a boundary; T K of them are used)
    ws = scratch(lib.b200q_grouped_mm_workspace_bytes(T, E, N, K, 1))
    run_threads(lambda i, y: bound(lib.b200q_grouped_mm, ptr(xs[i]), ptr(w), ptr(n), 8, ptr(y), _lib.BF16, T, E, N, K, 1, ptr(ws), ws.numel(), None), (T, N))


@pytest.mark.parametrize("n", (6, 64))
def test_gather_qmm(n):
    """Few rows and many, over the sorted pairs in scratch; a routing per thread."""
    lib, E, N, K, g, bits = _lib.load(), 4, 256, 256, 64, 4
    w, s, b = mb.quantize(torch.randn(E, N, K, device="cuda").bfloat16(), g, bits)
    x = torch.randn(n, K, device="cuda").bfloat16()
    lhs = torch.arange(n, dtype=torch.int32, device="cuda")
    rhs = (torch.arange(n, device="cuda") * 5 // 3 + torch.arange(THREADS, device="cuda")[:, None]).remainder(E).to(torch.int32)
    ws = scratch(lib.b200q_gather_qmm_workspace_bytes(_lib.BF16, n, n, E, 1, N, K, g, bits, 1))
    run_threads(lambda i, y: bound(lib.b200q_gather_qmm, ptr(x), ptr(w), ptr(s), ptr(b), ptr(lhs), ptr(rhs[i]), n, ptr(y), _lib.BF16, n, E, 1, N, K, g,
                                   bits, 1, 0, ptr(ws), ws.numel(), None), (n, N))
