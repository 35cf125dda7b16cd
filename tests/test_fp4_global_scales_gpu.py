"""nvfp4 products whose global scales multiply to more, or less, than fp32 holds, although the scaled sums are in its range."""
import numpy as np
import pytest
import torch

import fp4_plain as plain
import mlx_b200 as mb
from mlx_b200 import ops

pytestmark = pytest.mark.gpu


def u32(v):
    return torch.from_numpy(v.view(np.int32)).view(torch.uint32).cuda()


@pytest.mark.parametrize("T", (1, 8, 40))
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("gx,gw", ((2.0 ** 70, 2.0 ** 70), (2.0 ** 100, 2.0 ** 27), (2.0 ** -90, 2.0 ** -62)))
def test_nvfp4_global_scales_far_from_one(T, dtype, gx, gw):
    """What the two global scales multiply to need not be a fp32 number: zeros stay zeros, and what is in range is exact."""
    N, K = 48, 128
    codes = np.zeros((N, K), dtype=np.uint8)
    codes[1::2, 3] = 1                                    # 1/2
    scales = np.zeros((N, K // 16), dtype=np.uint8)
    scales[:, 0] = 1 if gx * gw > 1 else 0x7E             # 2^-9 or 448
    x = torch.zeros(T, K, device="cuda", dtype=dtype)
    # (x / gx is 2^-7: scale 2^-9, code 4; or, where everything is small, 448 * 4)
    x[:, 3] = gx * (2.0 ** -7 if gx * gw > 1 else 1792.0)
    one = lambda v: torch.tensor([v], device="cuda")
    y = mb.qqmm(x, u32(plain.pack(codes)), torch.from_numpy(scales).cuda(), mode="nvfp4", global_scale_x=one(gx), global_scale_w=one(gw))
    xq, sx = mb.quantize(x, mode="nvfp4", global_scale=one(gx))
    xv = plain.values(plain.unpack(plain.u32(xq)), sx.cpu().numpy(), "nvfp4", gx)
    with np.errstate(over="ignore", under="ignore"):
        ref = torch.from_numpy((xv @ plain.values(codes, scales, "nvfp4", gw).T).astype(np.float32)).to(dtype)
    assert torch.equal(y.cpu(), ref)
    ops.check_status()


@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("T,N,K", ((3, 130, 640), (40, 132, 256), (30, 200, 16384), (300, 513, 96)))
@pytest.mark.parametrize("gx,gw", ((0.0137, 3.1e-4), (1.7e-3, 0.9)))
def test_nvfp4_global_scales_that_are_no_powers_of_two(T, N, K, dtype, gx, gw):
    """Few rows, whole tiles, cut ones and odd widths; one scale, and one per expert."""
    for each in (False, True):
        E = 3 if each else 1
        g = torch.Generator("cuda").manual_seed(T)
        x, w = torch.randn(T, K, generator=g, device="cuda").to(dtype), torch.randn(E, N, K, generator=g, device="cuda") * 0.05
        sx, sw = torch.tensor([gx], device="cuda"), torch.tensor([gw, gw * 1.3, gw * 0.7][:E], device="cuda")
        (xq, xs), (wq, ws) = mb.quantize(x, mode="nvfp4", global_scale=sx), mb.quantize(w, mode="nvfp4", global_scale=sw)
        if each:
            n = [T // 3, 0, T - T // 3]
            y = mb.grouped_qqmm(x, wq, ws, torch.tensor(n, device="cuda"), mode="nvfp4", global_scale_x=sx, global_scale_w=sw)
        else:
            n = [T]
            y = mb.qqmm(x, wq[0], ws[0], mode="nvfp4", global_scale_x=sx, global_scale_w=sw)
        xv = plain.values(plain.unpack(plain.u32(xq)), xs.cpu().numpy(), "nvfp4", float(sx))
        wv = plain.values(plain.unpack(plain.u32(wq)), ws.cpu().numpy(), "nvfp4") * plain.f64(sw)[:, None, None]
        ref, mass = plain.grouped(xv, wv, n, True), plain.grouped(np.abs(xv), np.abs(wv), n, True)
        # (plain.allowed holds one factor; the product of the scales is rounded once more)
        room = plain.allowed(ref, mass, K, dtype) + 2.0 ** -24 * np.abs(ref) * 1.01
        assert (np.abs(plain.f64(y) - ref) <= room).all()
    ops.check_status()


@pytest.mark.parametrize("each", (False, True))
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("T,N,K", ((20, 48, 128), (20, 45, 16384), (300, 257, 64)))
def test_far_global_scales_through_tiles_that_are_cut_or_not(T, N, K, dtype, each):
    """x and its global scale times 2^70, the weights' scale 2^60 for 2^-70: the result times 2^200, bit for bit (the scales' product, 2^130,
    is no fp32 number; values of 2^-8 keep the result in range)."""
    E = 2 if each else 1
    g = torch.Generator("cuda").manual_seed(N)
    x, w = (torch.randn(T, K, generator=g, device="cuda") / 256).to(dtype), torch.randn(E, N, K, generator=g, device="cuda") / 256
    wq, ws = mb.quantize(w, mode="nvfp4")
    n = torch.tensor([T // 2, T - T // 2], device="cuda")

    def product(x, sx, sw):
        sx, sw = torch.tensor([sx], device="cuda"), torch.full((E,), sw, device="cuda")
        if each:
            return mb.grouped_qqmm(x, wq, ws, n, mode="nvfp4", global_scale_x=sx, global_scale_w=sw)
        return mb.qqmm(x, wq[0], ws[0], mode="nvfp4", global_scale_x=sx, global_scale_w=sw)

    near, far = product(x, 1.0, 2.0 ** -70), product(x * 2.0 ** 70, 2.0 ** 70, 2.0 ** 60)
    assert (near != 0).float().mean() > 0.9 and torch.isfinite(far).all()
    assert torch.equal(far, near * 2.0 ** 100 * 2.0 ** 100)
    ops.check_status()
