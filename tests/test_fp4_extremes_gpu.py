"""mxfp4 products of few rows whose scales multiply to more, or less, than fp32 holds, although the scaled sums are in its range."""
import numpy as np
import pytest
import torch

import fp4_plain as plain
import mlx_b200 as mb
from mlx_b200 import ops

pytestmark = pytest.mark.gpu


def u32(v):
    return torch.from_numpy(v.view(np.int32)).view(torch.uint32).cuda()


@pytest.mark.parametrize("T", (1, 8))
def test_mxfp4_scales_far_apart(T):
    """Scale bytes from elsewhere against large and small x: a group's sum of 0, 1/4 or 24 times both scales, which is exact wherever
    fp32 has the number; the product of the scales alone may pass its range."""
    K = 128
    for x_exp, w_exps in ((40, (-127, -100, 80, 85, 90, 91)), (100, (-127, 0, 20, 24, 30, 31)), (124, (-127, -3, 0, 6, 7)),
                          (-40, (-108, -107, -80, 0, 127)), (-120, (-28, -27, -4, 0, 120, 127))):
        codes, scales, row = np.zeros((16, K), dtype=np.uint8), np.full((16, K // 32), 254, dtype=np.uint8), 1
        for e in w_exps:
            for at, code in ((40, 1), (41, 15)):    # 1/2 times x's 1/2, -6 times x's 4
                if at == 40 or x_exp - 2 + e < 120:
                    codes[row, at], scales[row, 1] = code, e + 127
                    row += 1
        x = torch.zeros(T, K, device="cuda")
        x[:, 41], x[:, 40] = 2.0 ** x_exp, 2.0 ** (x_exp - 3)      # scale 2^(x_exp - 2)
        y = plain.f64(mb.qqmm(x, u32(plain.pack(codes)), torch.from_numpy(scales).cuda(), mode="mxfp4"))
        ref = (plain.f64(x) @ plain.values(codes, scales, "mxfp4").T).astype(np.float32).astype(np.float64)
        assert np.isfinite(ref).all() and (ref[:, 0] == 0).all()
        np.testing.assert_array_equal(y, ref)
    ops.check_status()


@pytest.mark.parametrize("sizes", (None, [3, 0, 5]))
def test_mxfp4_scales_with_x(sizes):
    """Times a power of two in x or in the weights' scale bytes, the result is times it too, bit for bit, whichever way the two scales
    are applied; x has a group of zeros, and one row a NaN."""
    T, N, K, E = 8, 48, 384, 1 if sizes is None else len(sizes)
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(T, K, generator=g, device="cuda")
    x[2, 64:96], x[5, 200] = 0, float("nan")
    w, s = mb.quantize(torch.randn(E, N, K, generator=g, device="cuda"), mode="mxfp4")
    n = None if sizes is None else torch.tensor(sizes, device="cuda")

    def product(x, s):
        return mb.qqmm(x, w[0], s[0], mode="mxfp4") if n is None else mb.grouped_qqmm(x, w, s, n, mode="mxfp4")

    ref = product(x, s)
    assert torch.isnan(ref[5]).all() and torch.isfinite(ref[[0, 1, 2, 3, 4, 6, 7]]).all()
    for k in (-60, -21, -20, -19, -14, -13, -12, -11, -10, -9, -1, 3, 4, 5, 6, 7, 8, 9, 40, 90):
        y = product(x * 2.0 ** k, s)
        assert torch.equal(torch.nan_to_num(y, 7.0), torch.nan_to_num(ref * 2.0 ** k, 7.0)), k
        if k < 60:
            y = product(x * 2.0 ** k, (s.int() - k).to(torch.uint8))
            assert torch.equal(torch.nan_to_num(y, 7.0), torch.nan_to_num(ref, 7.0)), k
