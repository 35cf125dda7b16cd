"""Refusals of the routing, of the rows' exchange and of the adapters: errors before any device work, on the host alone."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import _lib, grad


def refused(f, *a, error=ValueError, **kw):
    with pytest.raises(error):
        f(*a, **kw)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("f", (mb.route_experts, grad.route_experts))
def test_route_experts(f):
    x = torch.zeros(3, 8)
    refused(f, x, 2, error=RuntimeError)           # no CPU fallback
    for kw in (dict(top=0), dict(top=9), dict(scoring="relu"), dict(groups=3), dict(groups=0), dict(groups=2, top_groups=3), dict(groups=2, top_groups=0),
               dict(groups=4, top_groups=1, top=3), dict(group_best=3), dict(bias=torch.zeros(7)), dict(bias=torch.zeros(8, dtype=torch.int32)),
               dict(bias=torch.zeros(1, 8))):
        refused(f, x, **{"top": 2, **kw})
    refused(f, x.to(torch.int32), 2)
    refused(f, x.double(), 2)
    refused(f, torch.zeros(3, 0), 1)
    refused(f, torch.tensor(1.0), 1)
    refused(f, x, 1.5, error=TypeError)


def test_route_dlogits():
    refused(mb.route_dlogits, torch.zeros(3, 2), torch.zeros(3, 8), i32(3, 2), error=RuntimeError)
    refused(mb.route_dlogits, torch.zeros(3, 2), torch.zeros(3, 8), i32(3, 2).long())
    refused(mb.route_dlogits, torch.zeros(3, 2), torch.zeros(4, 8), i32(3, 2))
    refused(mb.route_dlogits, torch.zeros(3, 1), torch.zeros(3, 8), i32(3, 2))
    refused(mb.route_dlogits, torch.zeros(3, 2), torch.zeros(3, 8), i32(3, 2), "relu")


def test_rows():
    r = mb.Routing(torch.zeros(3, 2), i32(3, 2), i32(8), i32(3, 2), i32(6))
    for d, c in ((mb.dispatch_rows, mb.combine_rows), (grad.dispatch_rows, grad.combine_rows)):
        refused(d, bf(3, 4), r, error=RuntimeError)
        refused(c, bf(6, 4), r, error=RuntimeError)
        refused(d, bf(2, 4), r)
        refused(d, i32(3, 4), r)
        refused(d, bf(3, 4).double(), r)
        refused(d, bf(3, 4), r._replace(places=r.places.long()))
        refused(d, bf(3, 4), r._replace(order=i32(5)))
        refused(c, bf(5, 4), r)
        refused(c, bf(3, 2, 4), r)
        refused(c, bf(6, 4), r._replace(weights=torch.zeros(3, 1)))
        refused(c, bf(6, 4), r._replace(weights=i32(3, 2)))
    refused(mb.combine_rows_grad, bf(3, 4), bf(6, 4), r, error=RuntimeError)
    refused(mb.combine_rows_grad, bf(3, 5), bf(6, 4), r)
    refused(mb.combine_rows_grad, bf(3, 4).float(), bf(6, 4), r)


def test_adapters():
    refused(mb.group_rows, torch.zeros(3, dtype=torch.int64), 2, error=RuntimeError)
    refused(mb.group_rows, torch.zeros(3), 2)
    refused(mb.group_rows, torch.zeros(3, dtype=torch.bool), 2)
    refused(mb.group_rows, torch.zeros(3, dtype=torch.int64), -1)
    n = _lib.load().b200q_group_rows_tiles(5, 2)
    g = mb.RowGroups(i32(2), i32(3), i32(5), i32(n, 4))
    args = dict(y=bf(5, 8), x=bf(5, 16), a=bf(2, 4, 16), b=bf(2, 8, 4), groups=g)
    for f in (mb.add_adapters, grad.add_adapters):
        refused(f, **args, error=RuntimeError)
        for kw in (dict(x=bf(5, 16).float()), dict(y=bf(5, 8).half()), dict(a=bf(4, 16)), dict(b=bf(2, 4, 8)), dict(x=bf(4, 16)), dict(x=bf(5, 17)),
                   dict(y=bf(5, 9)), dict(a=bf(3, 4, 16)), dict(groups=g._replace(sizes=i32(3))), dict(groups=g._replace(order=i32(4))),
                   dict(groups=g._replace(order=i32(5).long())), dict(groups=g._replace(tiles=i32(n + 1, 4))), dict(groups=g._replace(starts=i32(2))),
                   dict(scales=torch.zeros(3)), dict(scales=i32(2))):
            refused(f, **{**args, **kw})
    refused(mb.add_adapters_grad, bf(5, 8), bf(5, 16), bf(2, 4, 16), bf(2, 8, 4), g, bf(5, 2, 16), error=RuntimeError)


def test_the_c_abi_refuses_before_any_cuda_call():
    lib = _lib.load()
    d, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4097)
    bad, ws_err, uns = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_WORKSPACE, _lib.ERR_UNSUPPORTED

    def route(logits=d, dtype=_lib.F32, T=4, E=8, top=2, scoring=0, groups=1, top_groups=1, best=1, ws=d, n=1 << 30, sizes=d):
        return lib.b200q_route(logits, dtype, T, E, top, scoring, None, groups, top_groups, best, 0, 1.0, d, d, sizes, d, d, ws, n, None)

    assert all(route(**kw) == bad for kw in (dict(logits=None), dict(dtype=7), dict(T=-1), dict(E=0), dict(top=0), dict(top=9), dict(scoring=2), dict(groups=3),
                                             dict(top_groups=2), dict(groups=4, top=3), dict(best=0), dict(sizes=None)))
    assert all(route(**kw) == uns for kw in (dict(E=1025), dict(E=64, top=33), dict(E=128, groups=64, top_groups=2), dict(T=1 << 31)))
    assert lib.b200q_route_workspace_bytes(4, 8, 2) == 0 and lib.b200q_route_workspace_bytes(4096, 8, 2) > 0
    assert route(T=4096, ws=None) == route(T=4096, n=8) == route(T=4096, ws=odd) == ws_err
    dl = lambda dw=d, dtype=_lib.F32, top=2, T=4: lib.b200q_route_dlogits(dw, d, dtype, d, T, 8, top, 0, 0, 1.0, d, None)
    assert dl(dw=None) == dl(dtype=5) == dl(top=9) == dl(T=-1) == bad and dl(T=0) == 0
    rows = lambda x=d, dtype=_lib.BF16, T=4, top=2, D=8: lib.b200q_dispatch_rows(x, dtype, T, top, D, d, d, d, None)
    assert rows(x=None) == rows(x=odd) == rows(dtype=3) == rows(T=-1) == rows(top=-1) == rows(D=-1) == bad
    assert rows(T=1 << 31) == rows(T=1 << 30, top=4) == rows(D=1 << 31) == uns and rows(T=0) == rows(top=0) == rows(D=0) == 0
    back = lambda y=d, dtype=_lib.BF16, out=d: lib.b200q_combine_rows(y, dtype, 4, 2, 8, d, d, out, None)
    assert back(y=None) == back(out=None) == back(y=odd) == back(dtype=9) == bad
    both = lambda dy=d, y=d, w=d, dys=d, dw=d: lib.b200q_combine_rows_grad(dy, y, _lib.F32, 4, 2, 8, d, d, w, dys, dw, None)
    assert both(dy=None) == both(y=None) == both(w=None) == both(dys=odd) == bad and both(dys=None, dw=None) == 0
    group = lambda ids=d, nb=8, T=4, n=3, ws=d, have=1 << 30, tiles=d: lib.b200q_group_rows(ids, nb, T, n, d, d, d, tiles, ws, have, None)
    assert group(ids=None) == group(nb=2) == group(ids=odd) == group(T=-1) == group(n=-1) == group(tiles=None) == group(tiles=ctypes.c_void_p(4104)) == bad
    assert group(n=4097) == group(T=(1 << 31) - 1) == uns and group(ws=None, T=5000) == group(have=4, T=5000) == ws_err
    add = lambda y=d, x=d, dtype=_lib.BF16, T=4, L=2, N=8, K=16, r=4, h=d, tiles=d, out=d: lib.b200q_add_adapters(
        y, x, d, d, dtype, T, L, N, K, r, d, tiles, None, h, out, None)
    assert add(y=None) == add(x=None) == add(h=None) == add(x=odd) == add(dtype=_lib.F32) == add(T=-1) == add(r=-1) == add(tiles=ctypes.c_void_p(4104)) == bad
    assert add(L=4097) == add(N=(1 << 24) + 1) == add(r=4097) == add(T=1 << 31) == uns
    assert add(T=0) == add(N=0) == add(L=0) == add(r=0) == 0      # (out is y: nothing to copy)
    g = lambda dy=d, x=d, a=d, b=d, h=d, g=d, dx=d, da=d, db=d, dtype=_lib.F16: lib.b200q_add_adapters_grad(
        dy, x, a, b, dtype, 4, 2, 8, 16, 4, d, d, d, None, h, g, dx, da, db, None)
    assert g(dy=None) == g(x=None) == g(a=None) == g(b=None) == g(h=None) == g(g=None) == g(dtype=_lib.F32) == g(dx=odd) == bad
    assert g(dx=None, da=None, db=None, g=None) == 0


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_the_cpp_shim_compiles_and_refuses(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe, libdir = str(tmp_path / "check"), os.path.dirname(_lib.LIB_PATH)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(root, "include"), os.path.join(root, "tests", "routing_shim_check.cpp"), "-o", exe,
                    "-L", libdir, "-lb200q", f"-Wl,-rpath,{libdir}"], check=True, capture_output=True, text=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and "SHIM-OK" in res.stdout, res.stdout + res.stderr
