"""Decode products of different widths from several host threads at once, straight into the library: each kernel keeps the shared memory that its largest call needs."""
import ctypes
import threading

import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import _lib

pytestmark = pytest.mark.gpu
CALLS = 1500


def ptr(t):
    return ctypes.c_void_p(t.data_ptr())


def product(M, N, K, bits, transpose, dtype):
    lib, code = _lib.load(), {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}[dtype]
    g = torch.Generator("cuda").manual_seed(K)
    w, s, b = mb.quantize(torch.randn((N, K) if transpose else (K, N), generator=g, device="cuda").to(dtype), 64, bits)
    x, y = torch.randn((M, K), generator=g, device="cuda").to(dtype), torch.empty((M, N), dtype=dtype, device="cuda")
    ws = torch.zeros(lib.b200q_qmm_workspace_bytes(code, 1, M, N, K, 64, bits, transpose), dtype=torch.uint8, device="cuda")
    values = (ptr(x), ptr(w), ptr(s), ptr(b), ptr(y), code, 1, M, N, K, 64, bits, transpose, 0, ptr(ws), ws.numel(), None)
    args = [t(v) if not isinstance(v, t) else v for t, v in zip(lib.b200q_qmm.argtypes, values)]
    # where warps add their parts in any order (transpose=0): 8 roundings of 2^-24 of the terms' magnitudes, twice, then one of the type each
    far = 0 if transpose else 2.0 ** -20 * (x.double().abs() @ mb.dequantize(w, s, b, 64, bits).double().abs())
    return y, lambda: lib.b200q_qmm(*args), far, (x, w, s, b, ws)


@pytest.mark.parametrize("M,N,bits,transpose,dtype,Ks", ((1, 512, 4, 1, torch.bfloat16, (512, 2048, 8192, 12288)), (8, 512, 8, 1, torch.float16, (1024, 4096, 8192, 2048)),
                                                         (16, 512, 4, 1, torch.bfloat16, (1024, 4096, 8192, 2048)), (12, 512, 2, 1, torch.bfloat16, (1024, 4096, 8192, 2048)),
                                                         (1, 9472, 4, 0, torch.bfloat16, (512, 2048, 16384, 32768))))
def test_threads(M, N, bits, transpose, dtype, Ks):
    jobs = [product(M, N, K, bits, transpose, dtype) for K in Ks]
    for _, call, _, _ in jobs:
        _lib.check(call())
    torch.cuda.synchronize()
    refs = [y.clone() for y, *_ in jobs]
    codes, gate = [0] * len(jobs), threading.Barrier(len(jobs))

    def work(i):
        gate.wait()
        for _ in range(CALLS):
            codes[i] |= jobs[i][1]()

    ts = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    [t.start() for t in ts]
    [t.join() for t in ts]
    torch.cuda.synchronize()
    assert codes == [0] * len(jobs)
    for (y, _, far, _), ref in zip(jobs, refs):
        assert torch.equal(y, ref) if transpose else ((y.double() - ref.double()).abs() <= far + torch.finfo(dtype).eps * ref.double().abs()).all()
