"""Pointers that are not on their elements' boundaries, which kernels would fault on, are refused by the routing, row and adapter calls before any CUDA call."""
import ctypes

import pytest

from mlx_b200 import _lib

AT = 4096
SIZES = {_lib.F32: 4, _lib.F16: 2, _lib.BF16: 2}


def each(call, pointers, off):
    """call(**{name: address}) with every pointer on its boundary but one; off[name]: its element's bytes."""
    for name in pointers:
        args = {n: ctypes.c_void_p(AT) for n in pointers}
        args[name] = ctypes.c_void_p(AT + off.get(name, 4) // 2)
        assert call(**args) == _lib.ERR_INVALID_ARGUMENT, name


@pytest.mark.parametrize("dtype", tuple(SIZES))
@pytest.mark.parametrize("T", (4, 4096))
def test_route(dtype, T):
    lib, ws = _lib.load(), ctypes.c_void_p(AT)
    each(lambda logits, bias, weights, experts, sizes, places, order: lib.b200q_route(
        logits, dtype, T, 8, 2, 0, bias, 1, 1, 1, 0, 1.0, weights, experts, sizes, places, order, ws, 1 << 30, None),
        ("logits", "bias", "weights", "experts", "sizes", "places", "order"), {"logits": SIZES[dtype]})
    each(lambda dw, logits, experts, dlogits: lib.b200q_route_dlogits(dw, logits, dtype, experts, T, 8, 2, 0, 0, 1.0, dlogits, None),
         ("dw", "logits", "experts", "dlogits"), {"logits": SIZES[dtype], "dlogits": SIZES[dtype]})
    assert lib.b200q_route(None, dtype, 0, 8, 2, 0, None, 1, 1, 1, 0, 1.0, None, None, ctypes.c_void_p(AT + 2), None, None, None, 0, None) == _lib.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("dtype", tuple(SIZES))
def test_rows(dtype):
    lib, n = _lib.load(), SIZES[dtype]
    each(lambda x, places, order, xs: lib.b200q_dispatch_rows(x, dtype, 4, 2, 8, places, order, xs, None), ("x", "places", "order", "xs"), {"x": n, "xs": n})
    each(lambda y, places, weights, out: lib.b200q_combine_rows(y, dtype, 4, 2, 8, places, weights, out, None), ("y", "places", "weights", "out"), {"y": n, "out": n})
    each(lambda dy, y, places, order, weights, dys, dw: lib.b200q_combine_rows_grad(dy, y, dtype, 4, 2, 8, places, order, weights, dys, dw, None),
         ("dy", "y", "places", "order", "weights", "dys", "dw"), {"dy": n, "y": n, "dys": n})
    assert lib.b200q_combine_rows_grad(None, None, dtype, 4, 2, 0, None, None, None, None, ctypes.c_void_p(AT + 2), None) == _lib.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("T", (4, 5000))
def test_group_rows(T):
    lib = _lib.load()
    for nb in (4, 8):
        each(lambda ids, sizes, starts, order, tiles: lib.b200q_group_rows(ids, nb, T, 3, sizes, starts, order, tiles, ctypes.c_void_p(AT), 1 << 30, None),
             ("ids", "sizes", "starts", "order", "tiles"), {"ids": nb, "tiles": 16})
    assert lib.b200q_group_rows(None, 4, 0, 3, ctypes.c_void_p(AT), ctypes.c_void_p(AT + 2), None, None, None, 0, None) == _lib.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("dtype", (_lib.F16, _lib.BF16))
def test_adapters(dtype):
    lib = _lib.load()
    sizes = {n: 2 for n in ("y", "x", "a", "b", "out", "dy", "dx", "da", "db")} | {n: 16 for n in ("tiles", "h", "g")}
    each(lambda y, x, a, b, order, tiles, scales, h, out: lib.b200q_add_adapters(y, x, a, b, dtype, 4, 2, 8, 16, 4, order, tiles, scales, h, out, None),
         ("y", "x", "a", "b", "order", "tiles", "scales", "h", "out"), sizes)
    each(lambda dy, x, a, b, order, starts, tiles, scales, h, g, dx, da, db: lib.b200q_add_adapters_grad(
        dy, x, a, b, dtype, 4, 2, 8, 16, 4, order, starts, tiles, scales, h, g, dx, da, db, None),
        ("dy", "x", "a", "b", "order", "starts", "tiles", "scales", "h", "g", "dx", "da", "db"), sizes)
