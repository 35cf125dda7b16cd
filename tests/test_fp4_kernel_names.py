"""Which kernel a 4-bit product takes, and both of them on either side of the line between them."""
import pytest
import torch

import mlx_b200 as mb

FEW, TILES = "fp4_rows", "grouped_tc"
MODES = ("mxfp4", "nvfp4")


@pytest.mark.parametrize("mode", MODES)
def test_where_the_kernel_for_few_rows_begins_and_ends(mode):
    name = lambda *a, **kw: mb.qqmm_kernel_name(*a, mode=mode, **kw)
    for T in range(1, 9):
        assert name(T, 100, 640) == FEW
    assert name(9, 100, 640) == name(16, 300, 1056 // 32 * 32) == TILES
    assert name(1, 15, 128) == TILES and name(1, 16, 128) == FEW       # a tile's rows
    assert name(1, 64, 128 + 32) == TILES and name(1, 64, 256) == FEW  # whole 128s of K
    assert name(1, 4096, 4096) == FEW and name(1, 14336, 4096) == FEW and name(1, 28672, 8192) == TILES
    assert name(8, 11424, 4096) == FEW and name(8, 11440, 4096) == TILES                                  # the estimate, dense
    assert name(8, 200, 128, experts=5) == FEW and name(9, 200, 128, experts=5) == TILES
    assert name(4, 5024, 4096, experts=4) == FEW and name(4, 5040, 4096, experts=4) == TILES              # and grouped
    assert name(4, 5024, 4096, experts=400) == FEW                                                        # (rows bound the experts that count)
    assert name(3, 48, 20608) == (TILES if mode == "mxfp4" else FEW)                                      # x and its scales in shared memory
    assert name(1, 64, 100) == name(-1, 64, 128) == name(1, 64, 128, experts=5000) == "invalid"


@pytest.mark.parametrize("mode", ("affine", "mxfp8", "other"))
def test_other_modes(mode):
    with pytest.raises((NotImplementedError, ValueError)):
        mb.qqmm_kernel_name(1, 64, 128, mode=mode)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("T,N,K,kernel", ((8, 11424, 4096, FEW), (8, 11440, 4096, TILES), (1, 14336, 4096, FEW), (1, 15360, 4608, TILES)))
def test_both_sides(T, N, K, kernel, mode):
    from test_fp4_gpu import check_qqmm

    assert mb.qqmm_kernel_name(T, N, K, mode=mode) == kernel
    a = check_qqmm(T, N, K, mode, "bf16")
    assert torch.equal(a, check_qqmm(T, N, K, mode, "bf16"))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("sizes,N,kernel", (([2, 0, 1, 1], 5024, FEW), ([2, 0, 1, 1], 5040, TILES)))
def test_both_sides_grouped(sizes, N, kernel, mode):
    from test_fp4_gpu import check_qqmm

    assert mb.qqmm_kernel_name(sum(sizes), N, 4096, mode=mode, experts=len(sizes)) == kernel
    check_qqmm(sum(sizes), N, 4096, mode, "bf16", sizes)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("T,N,K", ((1, 14, 256), (1, 15, 28672), (2, 8, 65536), (4, 256, 28640), (9, 4096, 4096), (16, 640, 16384)))
def test_single_rows_and_cut_tiles_of_the_tensor_core_kernel(T, N, K, mode):
    """Sizes that the kernel for few rows does not take: one row, and few tiles of long rows, which are cut."""
    from test_fp4_gpu import check_qqmm

    assert mb.qqmm_kernel_name(T, N, K, mode=mode) == TILES
    a = check_qqmm(T, N, K, mode, "bf16")
    assert torch.equal(a, check_qqmm(T, N, K, mode, "bf16"))
