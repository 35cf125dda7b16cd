"""The microscaled 4-bit modes on the GPU: quantize and dequantize code for code, qqmm and grouped_qqmm against 64 bits."""
import numpy as np
import pytest
import torch

import fp4_plain as plain
import mlx_b200 as mb
from mlx_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MODES = ("mxfp4", "nvfp4")


def randn(seed, shape, dtype, std=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def scalar(v):
    return torch.tensor([v], dtype=torch.float32, device="cuda")


def same_codes(w, mode, G=None):
    wq, s = mb.quantize(w, mode=mode, global_scale=None if G is None else scalar(G))
    c, sc = plain.quantize(plain.f64(w), mode, G)
    assert wq.dtype == torch.uint32 and s.dtype == torch.uint8
    np.testing.assert_array_equal(s.cpu().numpy(), sc)
    np.testing.assert_array_equal(plain.u32(wq), plain.pack(c))
    return wq, s


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("shape", ((1, 32), (3, 64), (77, 2080), (2, 5, 96), (4100, 512)))
def test_quantize_gives_the_definition_s_codes(shape, dtype, mode):
    w = randn(1, shape, DTYPES[dtype], 0.02)
    same_codes(w, mode)
    same_codes(w * 50, mode, None if mode == "mxfp4" else 2.0 ** -7)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", tuple(DTYPES))
def test_quantize_of_edge_groups(dtype, mode):
    """Zeros, ties, values beyond 6, subnormal numbers, the type's largest and smallest, one NaN or infinity in a group."""
    dt = DTYPES[dtype]
    # (nvfp4 of 32-bit values: of 16 bits, for which the test's own arithmetic is the definition's)
    fi = torch.finfo(torch.float16 if mode == "nvfp4" and dtype == "f32" else dt)
    g = plain.GROUP[mode]
    rows = [torch.zeros(g)]
    rows.append(torch.tensor([6.0] + [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0] * 5)[:g])          # ties, positive
    rows.append(-rows[1])
    rows.append(torch.tensor([7.75] + [6.5, 7.0, -7.5, -0.0, 0.1] * 7)[:g])
    rows += [torch.full((g,), fi.max), torch.full((g,), -fi.tiny), torch.full((g,), fi.smallest_normal * 4)]
    rows.append(torch.tensor([fi.max, fi.tiny] * 16)[:g])
    for bad in (float("nan"), float("inf"), float("-inf")):
        r = torch.ones(g)
        r[g - 3] = bad
        rows.append(r)
    w = torch.cat(rows).reshape(1, -1).to(dt).cuda()
    if mode == "nvfp4" and dtype == "f32":
        w = w.to(torch.float16).float()
    wq, s = same_codes(w, mode)
    v = mb.dequantize(wq, s, mode=mode, dtype=torch.float32).reshape(-1, g)
    assert torch.isnan(v[-3:]).all() and torch.isfinite(v[:-3]).all()


def test_nvfp4_follows_its_definition_in_fp32_operation_by_operation():
    """Any global scale and 32-bit values: numpy's fp32 operations are the definition's."""
    for seed, G in ((1, 3.1e-5), (2, 0.7), (3, 1.9e4), (4, 1e-30), (5, 2.5e-39)):
        w = randn(seed, (64, 512), torch.float32, 0.02)
        wq, s = mb.quantize(w, mode="nvfp4", global_scale=scalar(G))
        v = w.cpu().numpy().reshape(64, 32, 16)
        G32 = np.float32(G)
        with np.errstate(all="ignore"):
            sc = plain.nearest_code(np.minimum((np.abs(v).max(-1) / (np.float32(6) * G32)).astype(np.float64), 448.0), plain.E4M3[:127])
            d = plain.E4M3[sc].astype(np.float32) * G32
            t = np.where(d[..., None] > 0, np.abs(v) / d[..., None], np.float32(0))
        c = plain.nearest_code(t.astype(np.float64), plain.E2M1) + 8 * np.signbit(v)
        np.testing.assert_array_equal(s.cpu().numpy(), sc.astype(np.uint8))
        np.testing.assert_array_equal(plain.unpack(plain.u32(wq)).reshape(c.shape), c)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", tuple(DTYPES))
def test_dequantize(dtype, mode):
    """Every code under every scale, rounded once from fp32."""
    dt = DTYPES[dtype]
    g = plain.GROUP[mode]
    scales = torch.arange(256 if mode == "mxfp4" else 128, dtype=torch.uint8, device="cuda").repeat_interleave(2)[None]   # all 16 codes: two groups of 16, or more
    codes = np.tile(np.arange(16, dtype=np.uint8), scales.numel() * g // 16)[None]
    wq = torch.from_numpy(plain.pack(codes).view(np.int32)).view(torch.uint32).cuda()
    G = None if mode == "mxfp4" else 0.37
    v = mb.dequantize(wq, scales, mode=mode, dtype=dt, global_scale=None if G is None else scalar(G))
    assert v.dtype == dt
    exact = plain.values(codes, scales.cpu().numpy(), mode)
    with np.errstate(all="ignore"):
        ref = exact.astype(np.float32) if G is None else exact.astype(np.float32) * np.float32(G)
    ref = torch.from_numpy(ref).to(dt)
    assert torch.equal(torch.nan_to_num(v.cpu().float(), nan=-7.0), torch.nan_to_num(ref.float(), nan=-7.0))
    assert mb.dequantize(wq, scales, mode=mode).dtype == torch.bfloat16


def test_stacks_strides_and_addresses():
    """A scale for the whole stack or one per matrix; views, transposes and storage that is not aligned."""
    w = randn(3, (3, 40, 64), torch.bfloat16, 0.5)
    G = torch.tensor([0.5, 1.0, 0.25], device="cuda")
    wq, s = mb.quantize(w, mode="nvfp4", global_scale=G)
    for e in range(3):
        a, b = mb.quantize(w[e], mode="nvfp4", global_scale=G[e:e + 1])
        assert torch.equal(a.view(torch.int32), wq[e].view(torch.int32)) and torch.equal(b, s[e])
    v = mb.dequantize(wq, s, mode="nvfp4", global_scale=G)
    assert torch.equal(v[1], mb.dequantize(wq[1], s[1], mode="nvfp4", global_scale=G[1:2]))
    flat = randn(4, (1 + 40 * 64,), torch.bfloat16)
    odd = flat[1:].reshape(40, 64)
    for view in (odd, odd.t().contiguous().t(), w[:, ::2], w.transpose(0, 1)[:, 1]):
        a, b = mb.quantize(view, mode="mxfp4")
        c, d = mb.quantize(view.clone(memory_format=torch.contiguous_format), mode="mxfp4")
        assert torch.equal(a.view(torch.int32), c.view(torch.int32)) and torch.equal(b, d)
    assert mb.quantize(torch.zeros(0, 32, device="cuda"), mode="mxfp4")[0].shape == (0, 4)
    assert mb.dequantize(*mb.quantize(torch.zeros(5, 0, device="cuda"), mode="mxfp4"), mode="mxfp4").shape == (5, 0)


def check_qqmm(T, N, K, mode, dtype, sizes=None, G=True, seed=1, scale_base=0):
    dt = DTYPES[dtype]
    E = 1 if sizes is None else len(sizes)
    x = randn(seed, (T, K), dt)
    w = randn(seed + 1, (E, N, K), torch.bfloat16, 0.02)
    gw = gx = None
    if mode == "nvfp4" and G:
        gx, gw = scalar(2.0 ** -9), torch.tensor([2.0 ** -(15 + e % 3) for e in range(E)], device="cuda")
    wq, s = mb.quantize(w, mode=mode, global_scale=gw)
    xq, sx = mb.quantize(x, mode=mode, global_scale=gx)
    if scale_base:   # scales off every boundary
        s = torch.cat((torch.zeros(scale_base, dtype=torch.uint8, device="cuda"), s.flatten()))[scale_base:].reshape(s.shape)
    if sizes is None:
        y = mb.qqmm(x, wq[0], s[0], mode=mode, global_scale_x=gx, global_scale_w=gw)
    else:
        y = mb.grouped_qqmm(x, wq, s, torch.tensor(sizes, device="cuda"), mode=mode, global_scale_x=gx, global_scale_w=gw)
    ops.check_status()
    assert y.shape == (T, N) and y.dtype == dt
    xv = plain.values(plain.unpack(plain.u32(xq)), sx.cpu().numpy(), mode, None if gx is None else gx.item())
    wv = plain.values(plain.unpack(plain.u32(wq)), s.cpu().numpy(), mode)
    if gw is not None:
        wv = wv * gw.cpu().numpy()[:, None, None]
    n = [T] if sizes is None else sizes
    ref, mass = plain.grouped(xv, wv, n, True), plain.grouped(np.abs(xv), np.abs(wv), n, True)
    err = np.abs(plain.f64(y) - ref)
    assert (err <= plain.allowed(ref, mass, K, dt)).all(), (err / plain.allowed(ref, mass, K, dt)).max()
    return y


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", tuple(DTYPES))
@pytest.mark.parametrize("T,N,K", ((1, 256, 256), (1, 1, 32), (16, 300, 1056), (17, 129, 64), (63, 1000, 4096), (129, 40, 96),
                                   (255, 257, 544), (256, 512, 2048), (300, 640, 1024)))
def test_qqmm(T, N, K, mode, dtype):
    check_qqmm(T, N, K, mode, dtype)


@pytest.mark.parametrize("K", (16, 48, 80, 1008, 4112))
def test_qqmm_of_widths_that_end_inside_a_tile(K):
    """Rows of codes off 16-byte boundaries (odd groups of 16), rows of scales off every boundary."""
    check_qqmm(37, 200, K, "nvfp4", "bf16")
    check_qqmm(2, 130, K * 2, "mxfp4", "f16")
    check_qqmm(5, 130, K, "nvfp4", "f32", scale_base=3)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("T,N,K", ((1, 4096, 4096), (4, 256, 28672), (130, 256, 16384), (700, 2048, 512)))
def test_qqmm_over_cut_tiles_and_waves(T, N, K, mode):
    """Few tiles of long rows (cut, their parts added up), and several waves; the same bits every time."""
    a = check_qqmm(T, N, K, mode, "bf16")
    assert torch.equal(a, check_qqmm(T, N, K, mode, "bf16"))


def test_qqmm_shapes_streams_and_graphs():
    x = randn(1, (2, 3, 64), torch.bfloat16)
    w = randn(2, (96, 64), torch.bfloat16)
    wq, s = mb.quantize(w, mode="mxfp4")
    y = mb.qqmm(x, wq, s, mode="mxfp4")
    assert y.shape == (2, 3, 96)
    assert torch.equal(y[1, 2], mb.qqmm(x[1, 2], wq, s, mode="mxfp4"))
    assert torch.equal(y, mb.qqmm(x.transpose(0, 1).contiguous().transpose(0, 1), wq, s, mode="mxfp4"))
    assert mb.qqmm(x[:0], wq, s, mode="mxfp4").shape == (0, 3, 96)
    assert mb.qqmm(x, wq[:0], s[:0], mode="mxfp4").shape == (2, 3, 0)
    assert (mb.qqmm(x[..., :0], wq[:, :0], s[:, :0], mode="mxfp4") == 0).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(y, mb.qqmm(x, wq, s, mode="mxfp4"))
        graph = torch.cuda.CUDAGraph()
        xs = x.clone()
        with torch.cuda.graph(graph, stream=side):
            z = mb.qqmm(xs, wq, s, mode="mxfp4")
        for k in (1.0, -2.0):
            xs.copy_(x * k)
            graph.replay()
            side.synchronize()
            assert torch.equal(z, y * k)   # powers of two: the same codes
    ops.check_status()


def test_a_row_that_is_not_finite_is_nan_and_no_other():
    x = randn(1, (40, 256), torch.bfloat16)
    clean = x.clone()
    x[3, 17], x[20, 255], x[39, 0] = float("nan"), float("inf"), float("-inf")
    wq, s = mb.quantize(randn(2, (300, 256), torch.bfloat16), mode="nvfp4")
    y, ref = mb.qqmm(x, wq, s), mb.qqmm(clean, wq, s)
    bad = torch.tensor([3, 20, 39], device="cuda")
    assert torch.isnan(y[bad]).all()
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[bad] = False
    assert torch.equal(y[keep], ref[keep])


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", ("bf16", "f32"))
@pytest.mark.parametrize("sizes,N,K", (((0, 5, 0, 1, 12), 300, 512), ((1,), 16, 32), ((0, 0), 64, 64), ((300, 0, 17, 256), 257, 544),
                                       (tuple(range(40)), 128, 96), ((3,) * 300, 48, 64), ((700, 1), 512, 2080)))
def test_grouped_qqmm(sizes, N, K, mode, dtype):
    check_qqmm(max(1, sum(sizes)), N, K, mode, dtype, list(sizes))


def test_grouped_qqmm_skips_experts_without_rows():
    """The scales of an expert without rows may be anything."""
    x = randn(1, (9, 64), torch.bfloat16)
    wq, s = mb.quantize(randn(2, (3, 200, 64), torch.bfloat16), mode="mxfp4")
    sizes = torch.tensor([4, 0, 5], device="cuda")
    y = mb.grouped_qqmm(x, wq, s, sizes, mode="mxfp4")
    s[1] = 255
    assert torch.equal(y, mb.grouped_qqmm(x, wq, s, sizes, mode="mxfp4")) and torch.isfinite(y).all()


def test_grouped_qqmm_of_the_most_groups():
    """The table of 4096 groups leaves room for few stages and few scales."""
    E, N, K = 4096, 24, 1088
    sizes = [3 if e % 13 == 0 else (300 if e == 2000 else 0) for e in range(E)]
    check_qqmm(sum(sizes), N, K, "nvfp4", "bf16", sizes)
