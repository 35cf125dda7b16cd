"""4-bit products of up to 8 rows, which have a kernel of their own, around the sizes where it begins and ends."""
import numpy as np
import pytest
import torch

import fp4_plain as plain
import mlx_b200 as mb
from mlx_b200 import ops
from test_fp4_gpu import DTYPES, MODES, check_qqmm, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", tuple(DTYPES))
@pytest.mark.parametrize("T", (1, 2, 3, 7, 8, 9))
def test_rows(T, dtype, mode):
    check_qqmm(T, 100, 640, mode, dtype)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("N,K", ((15, 128), (16, 128), (17, 256), (31, 384), (33, 4096), (5000, 128), (4096, 4096), (2500, 2176), (48, 20608), (20000, 512)))
def test_tiles_halves_and_splits(N, K, mode):
    """The last tile begins earlier, the last piece of K has one half, one to sixteen warps share a tile, several rounds."""
    a = check_qqmm(3, N, K, mode, "bf16")
    assert torch.equal(a, check_qqmm(3, N, K, mode, "bf16"))


@pytest.mark.parametrize("mode", MODES)
def test_scales_and_x_off_their_boundaries(mode):
    for base in (1, 2, 4, 8):
        check_qqmm(4, 64, 256, mode, "bf16", scale_base=base)
    x, w = randn(1, (5 * 256 + 1,), torch.bfloat16), randn(2, (40, 256), torch.bfloat16)
    wq, s = mb.quantize(w, mode=mode)
    odd = x[1:].reshape(5, 256)
    assert torch.equal(mb.qqmm(odd, wq, s, mode=mode), mb.qqmm(odd.clone(), wq, s, mode=mode))


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("sizes", ((8,), (1,) * 8, (0, 3, 0, 0, 1, 4), (0,) * 70 + (2,) + (0,) * 600 + (5,) + (0,) * 29, (0, 0, 0)))
@pytest.mark.parametrize("N,K", ((16, 128), (45, 1152)))
def test_groups(N, K, sizes, mode):
    check_qqmm(max(1, sum(sizes)), N, K, mode, "f16", list(sizes))
    check_qqmm(8, N, K, mode, "bf16", list(sizes))   # rows of no group are zero


@pytest.mark.parametrize("sizes,kept", (([3, 9, 1], [3, 4, 0]), ([-3, 2, 1], [0, 2, 1]), ([2 ** 40, 1, 1], [7, 0, 0]), ([7, -2 ** 40, 2 ** 62], [7, 0, 0])))
def test_sizes_that_do_not_fit(sizes, kept):
    x = randn(1, (7, 128), torch.bfloat16)
    wq, s = mb.quantize(randn(2, (3, 50, 128), torch.bfloat16), mode="nvfp4")
    ops.check_status()
    y = mb.grouped_qqmm(x, wq, s, torch.tensor(sizes, device="cuda"))
    with pytest.raises(ops.DeviceStatusError) as e:
        ops.check_status()
    assert e.value.code == 9
    assert torch.equal(y, mb.grouped_qqmm(x, wq, s, torch.tensor(kept, device="cuda")))
    small = torch.tensor(kept, device="cuda", dtype=torch.int32)
    assert torch.equal(y, mb.grouped_qqmm(x, wq, s, small))
    ops.check_status()


@pytest.mark.parametrize("mode", MODES)
def test_what_is_not_finite_stays_in_its_row_and_column(mode):
    x, w = randn(1, (6, 384), torch.bfloat16), randn(2, (70, 384), torch.bfloat16)
    clean = mb.qqmm(x, *mb.quantize(w, mode=mode), mode=mode)
    x[2, 100], x[5, 383] = float("nan"), float("-inf")
    w[11, 5], w[69, 383] = float("inf"), float("nan")
    y = mb.qqmm(x, *mb.quantize(w, mode=mode), mode=mode)
    bad = torch.zeros(6, 70, dtype=torch.bool, device="cuda")
    bad[[2, 5]] = True
    bad[:, [11, 69]] = True
    assert torch.equal(torch.isnan(y), bad)
    assert torch.equal(y[~bad], clean[~bad])
    sizes = torch.tensor([2, 4], device="cuda")   # and in its group
    wq, s = mb.quantize(torch.stack((torch.full_like(w, float("nan")), torch.nan_to_num(w, 0, 0, 0))), mode=mode)
    z = mb.grouped_qqmm(torch.nan_to_num(x, 0, 0, 0), wq, s, sizes, mode=mode)
    assert torch.isnan(z[:2]).all() and torch.isfinite(z[2:]).all()


def test_every_e8m0_scale():
    """Codes and scales from elsewhere: 0 is 2^-127, 255 is NaN whatever the codes."""
    g = torch.Generator("cuda").manual_seed(3)
    N, K = 256, 256
    wq = torch.randint(0, 2 ** 31, (N, K // 8), generator=g, device="cuda", dtype=torch.int32).view(torch.uint32)
    s = torch.arange(256, device="cuda", dtype=torch.uint8)[:, None].expand(N, K // 32).contiguous()
    x = randn(1, (4, K), torch.float32)
    xq, sx = mb.quantize(x, mode="mxfp4")
    y = plain.f64(mb.qqmm(x, wq, s, mode="mxfp4"))
    assert np.isnan(y[:, 255]).all()
    xv = plain.values(plain.unpack(plain.u32(xq)), sx.cpu().numpy(), "mxfp4")
    wv = plain.values(plain.unpack(plain.u32(wq)), s.cpu().numpy(), "mxfp4")[:240]   # beyond, sums pass fp32's range
    ref, mass = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    assert (np.abs(y[:, :240] - ref) <= plain.allowed(ref, mass, K, torch.float32)).all()
