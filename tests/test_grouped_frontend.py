"""Refusals of the microscaled modes and the grouped products: ValueError before any device work, on the host alone."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import _lib, grad


def u32(*shape):
    return torch.zeros(shape, dtype=torch.int32).view(torch.uint32)


def u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def refused(f, *a, error=ValueError, **kw):
    with pytest.raises(error):
        f(*a, **kw)


def test_quantize_and_dequantize():
    for mode, g in (("mxfp4", 32), ("nvfp4", 16)):
        refused(mb.quantize, torch.zeros(4, 3 * g + 1), mode=mode)
        refused(mb.quantize, torch.zeros(g), mode=mode)
        refused(mb.quantize, torch.zeros(4, g, dtype=torch.int32), mode=mode)
        refused(mb.quantize, torch.zeros(4, 64), mode=mode, group_size=64)
        refused(mb.quantize, torch.zeros(4, 64), mode=mode, bits=8)
        refused(mb.dequantize, u32(4, g // 8), u8(4, 2), mode=mode)
        refused(mb.dequantize, u32(4, g // 8), torch.zeros(4, 1), mode=mode)
        refused(mb.dequantize, torch.zeros(4, g // 8), u8(4, 1), mode=mode)
        refused(mb.dequantize, u32(4, g // 8), u8(4, 1), torch.zeros(4, 1), mode=mode)          # no biases
        refused(mb.dequantize, u32(4, g // 8), u8(4, 1), mode=mode, dtype=torch.int32)
        refused(mb.quantize, torch.zeros(4, g), mode=mode, error=RuntimeError)                   # no CPU fallback
    one = torch.ones(1)
    refused(mb.quantize, torch.zeros(4, 64), mode="mxfp4", global_scale=one, error=(ValueError, RuntimeError))
    refused(mb.quantize, torch.zeros(4, 64), global_scale=one)                                   # affine
    refused(mb.dequantize, u32(4, 8), torch.zeros(4, 1), torch.zeros(4, 1), global_scale=one)
    refused(mb.quantize, torch.zeros(4, 64), mode="mxfp8", error=NotImplementedError)
    refused(mb.quantized_matmul, bf(2, 64), u32(4, 8), u8(4, 2), mode="mxfp4", error=NotImplementedError)
    refused(mb.gather_qmm, bf(2, 64), u32(4, 8), u8(4, 2), mode="nvfp4", error=NotImplementedError)


def test_qqmm():
    x, w, s = bf(3, 64), u32(5, 8), u8(5, 2)
    call = lambda x=x, w=w, s=s, error=ValueError, mode="mxfp4", **kw: refused(mb.qqmm, x, w, s, mode=mode, error=error, **kw)
    call(error=RuntimeError)                       # CPU tensors
    call(mode="nvfp4")                             # scales of another group size
    call(mode="affine", error=NotImplementedError)
    call(mode="mxfp8", error=NotImplementedError)
    call(mode="no such mode")
    call(x=bf(3, 32))
    call(x=torch.zeros(3, 64, dtype=torch.int8))
    call(x=torch.zeros(3, 64, dtype=torch.float64))
    call(w=u32(5, 8).view(torch.int32))
    call(s=torch.zeros(5, 2))
    call(s=u8(4, 2))
    call(w=u32(2, 5, 8), s=u8(2, 5, 2))            # a stack needs sizes
    call(bits=8)
    call(group_size=64)
    call(x=torch.tensor(1.0))


def test_grouped():
    x, w, n = bf(6, 16), bf(2, 8, 16), torch.tensor([2, 4])
    for f in (mb.grouped_mm, grad.grouped_mm):
        refused(f, x, w, n, error=RuntimeError)
        refused(f, x, w.float(), n)
        refused(f, x.float(), w.float(), n)        # 16 bits only
        refused(f, x, w.half(), n)
        refused(f, x, w, n, False)                 # the other layout's widths
        refused(f, x[0], w, n)
        refused(f, x, w[0], n)
    refused(mb.grouped_mm_dw, bf(6, 8), bf(5, 16), n)
    refused(mb.grouped_mm_dw, bf(6, 8).float(), x, n)
    refused(mb.grouped_mm_dw, bf(6, 8), x[None], n)
    refused(mb.grouped_mm_dw, bf(6, 8), x, n, error=RuntimeError)
    refused(mb.grouped_qqmm, bf(6, 64), u32(2, 8, 8), u8(2, 8, 2), n, mode="mxfp4", error=RuntimeError)
    refused(mb.grouped_qqmm, bf(6, 64), u32(8, 8), u8(8, 2), n, mode="mxfp4")
    refused(mb.grouped_qqmm, bf(1, 6, 64), u32(2, 8, 8), u8(2, 8, 2), n, mode="mxfp4")


def test_the_c_abi_refuses_before_any_cuda_call():
    lib = _lib.load()
    d, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4100)
    bad, ws_err, uns = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_WORKSPACE, _lib.ERR_UNSUPPORTED
    q = lambda dtype=_lib.BF16, rows=4, K=64, mode=_lib.MXFP4, g=None, per=1, wq=d: lib.b200q_fp4_quantize(d, dtype, rows, K, mode, g, per, wq, d, None)
    assert q(dtype=7) == q(K=40) == q(mode=2) == q(rows=-1) == q(g=d) == q(mode=_lib.NVFP4, g=d, per=0) == q(wq=odd) == bad
    assert q(rows=0) == q(K=0) == 0
    dq = lambda dtype=_lib.BF16, K=64, mode=_lib.NVFP4, wq=d: lib.b200q_fp4_dequantize(wq, d, mode, None, 1, dtype, 4, K, d, None)
    assert dq(dtype=3) == dq(K=24) == dq(mode=-1) == dq(wq=odd) == bad
    mm = lambda x=d, dtype=_lib.BF16, T=4, E=2, N=8, K=16, sizes=d, sb=8, ws=d, n=1 << 30: lib.b200q_grouped_mm(
        x, d, sizes, sb, d, dtype, T, E, N, K, 1, ws, n, None)
    assert mm(dtype=_lib.F32) == mm(T=-1) == mm(sizes=None) == mm(sb=2) == mm(x=odd) == mm(x=None) == bad
    assert mm(ws=None) == mm(n=1024) == mm(n=(1 << 30) + 8) == ws_err
    assert mm(E=4097) == mm(N=1 << 31) == uns
    assert mm(T=0) == mm(N=0) == 0
    need = lib.b200q_grouped_mm_workspace_bytes(4, 2, 8, 16, 1)
    assert need % 16 == 0 and lib.b200q_grouped_mm_workspace_bytes(4, 2, 8, 17, 1) > need     # rows of 34 bytes are copied
    dw = lambda dy=d, dtype=_lib.F16, E=2, ws=d, sizes=d: lib.b200q_grouped_mm_dw(dy, d, sizes, 4, d, dtype, 4, E, 8, 16, ws, 1 << 30, None)
    assert dw(dtype=_lib.F32) == dw(dy=None) == dw(dy=odd) == dw(sizes=None) == dw(E=-1) == bad
    assert dw(ws=None) == ws_err and dw(E=5000) == uns and dw(E=0) == 0
    qq = lambda wq=d, E=1, sizes=None, K=64, mode=_lib.MXFP4, gx=None, ws=d: lib.b200q_grouped_qqmm(
        d, wq, d, sizes, 8, d, _lib.BF16, 4, E, 8, K, mode, gx, None, 0, ws, 1 << 30, None)
    assert qq(E=2) == qq(wq=odd) == qq(K=33) == qq(mode=9) == qq(gx=d) == qq(wq=None) == bad
    assert qq(ws=None) == ws_err


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_the_cpp_shim_compiles_and_refuses(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe, libdir = str(tmp_path / "check"), os.path.dirname(_lib.LIB_PATH)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(root, "include"), os.path.join(root, "tests", "grouped_shim_check.cpp"), "-o", exe,
                    "-L", libdir, "-lb200q", f"-Wl,-rpath,{libdir}"], check=True, capture_output=True, text=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and "SHIM-OK" in res.stdout, res.stdout + res.stderr
