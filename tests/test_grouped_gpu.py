"""Products grouped by expert with ragged sizes, and their gradients, against 64 bits."""
import numpy as np
import pytest
import torch

import fp4_plain as plain
import mlx_b200 as mb
from mlx_b200 import grad, ops

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def randn(seed, shape, dtype, std=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def close(y, ref, mass, terms, dtype):
    err, ok = np.abs(plain.f64(y) - ref), plain.allowed(ref, mass, terms, dtype)
    assert (err <= ok).all(), (err / ok).max()


SIZES = ((5,), (0, 5, 0, 1, 12), (0, 0, 3), (64, 64), (63, 65, 1), (300, 0, 17, 256), (257, 15, 16), tuple(range(40)), (2,) * 300, (1000, 1, 24))


@pytest.mark.parametrize("dtype", tuple(DTYPES))
@pytest.mark.parametrize("transpose", (True, False))
@pytest.mark.parametrize("sizes", SIZES)
def test_grouped_mm_and_its_gradients(sizes, transpose, dtype):
    """Widths that are whole tiles, end inside one, and have rows off 16-byte boundaries; experts without rows; a row or many."""
    dt, T, E = DTYPES[dtype], sum(sizes), len(sizes)
    for N, K in ((256, 128), (300, 136), (77, 100), (130, 513)):
        if E > 50 and N != 77:
            continue
        x, w = randn(1, (T, K), dt), randn(2, (E, N, K) if transpose else (E, K, N), dt, 0.1)
        dy = randn(3, (T, N), dt)
        st = torch.tensor(sizes, device="cuda", dtype=torch.int32 if N == 77 else torch.int64)
        y = mb.grouped_mm(x, w, st, transpose)
        dx, dw = mb.grouped_mm(dy, w, st, not transpose), mb.grouped_mm_dw(dy, x, st, transpose)
        ops.check_status()
        X, W, D = plain.f64(x), plain.f64(w), plain.f64(dy)
        close(y, plain.grouped(X, W, sizes, transpose), plain.grouped(abs(X), abs(W), sizes, transpose), K, dt)
        close(dx, plain.grouped(D, W, sizes, not transpose), plain.grouped(abs(D), abs(W), sizes, not transpose), N, dt)
        close(dw, plain.grouped_dw(D, X, sizes, transpose), plain.grouped_dw(abs(D), abs(X), sizes, transpose), max(sizes), dt)
        assert dw.shape == w.shape and y.dtype == dx.dtype == dw.dtype == dt
        for e in range(E):
            if sizes[e] == 0:
                assert (dw[e] == 0).all()


@pytest.mark.parametrize("sizes,N,K", (((1,), 4096, 8192), ((3, 0, 2), 256, 28672), ((600, 424), 2048, 1024), ((4096,), 256, 256), ((150,), 512, 20000)))
def test_cut_tiles_and_waves(sizes, N, K):
    """Few tiles with long sums (cut, their parts added up) and several waves, in every direction; the same bits every time."""
    T, E = sum(sizes), len(sizes)
    x, w, dy = randn(1, (T, K), torch.bfloat16), randn(2, (E, N, K), torch.bfloat16, 0.1), randn(3, (T, N), torch.bfloat16)
    st = torch.tensor(sizes, device="cuda")
    X, W, D = plain.f64(x), plain.f64(w), plain.f64(dy)
    for f, ref, mass, terms in ((lambda: mb.grouped_mm(x, w, st), plain.grouped(X, W, sizes, True), plain.grouped(abs(X), abs(W), sizes, True), K),
                                (lambda: mb.grouped_mm(dy, w, st, False), plain.grouped(D, W, sizes, False), plain.grouped(abs(D), abs(W), sizes, False), N),
                                (lambda: mb.grouped_mm_dw(dy, x, st), plain.grouped_dw(D, X, sizes, True), plain.grouped_dw(abs(D), abs(X), sizes, True), T)):
        a = f()
        close(a, ref, mass, terms, torch.bfloat16)
        assert all(torch.equal(a, f()) for _ in range(3))
    ops.check_status()


def test_infinities_and_nans_stay_in_their_group():
    """An expert's rows and matrix do not reach another's results, where tiles of 16 k and of 256 rows overlap them: the masked rows
    of a tile are zeros in both operands."""
    sizes, N, K = [19, 30, 0, 15], 96, 72
    T = sum(sizes)
    x, dy = randn(1, (T, K), torch.bfloat16), randn(2, (T, N), torch.bfloat16)
    w = randn(3, (4, N, K), torch.bfloat16)
    st = torch.tensor(sizes, device="cuda")
    ref = mb.grouped_mm(x, w, st), mb.grouped_mm(dy, w, st, False), mb.grouped_mm_dw(dy, x, st)
    for bad in (float("nan"), float("inf")):
        x2, dy2, w2 = x.clone(), dy.clone(), w.clone()
        x2[19:49], dy2[19:49], w2[1] = bad, bad, bad
        y, dx, dw = mb.grouped_mm(x2, w2, st), mb.grouped_mm(dy2, w2, st, False), mb.grouped_mm_dw(dy2, x2, st)
        for a, r in ((y, ref[0]), (dx, ref[1])):
            assert torch.equal(a[:19], r[:19]) and torch.equal(a[49:], r[49:]) and not torch.isfinite(a[19:49]).any()
        assert torch.equal(dw[0], ref[2][0]) and torch.equal(dw[2:], ref[2][2:]) and not torch.isfinite(dw[1]).any()
    x2 = x.clone()
    x2[5, 3] = float("inf")   # one infinity: what its weight's sign says
    y = mb.grouped_mm(x2, w, st)
    assert torch.equal(torch.isinf(y).nonzero()[:, 0].unique().cpu(), torch.tensor([5]))
    assert torch.equal(torch.sign(y[5]), torch.sign(w[0, :, 3]))


def test_rows_that_belong_to_no_group():
    x, w = randn(1, (50, 64), torch.bfloat16), randn(2, (3, 33, 64), torch.bfloat16)
    st = torch.tensor([10, 0, 7], device="cuda")
    y = mb.grouped_mm(x, w, st)
    assert (y[17:] == 0).all() and torch.equal(y[:17], mb.grouped_mm(x[:17].contiguous(), w, st))
    dy = randn(3, (50, 33), torch.bfloat16)
    assert torch.equal(mb.grouped_mm_dw(dy, x, st), mb.grouped_mm_dw(dy[:17].contiguous(), x[:17].contiguous(), st))
    assert (mb.grouped_mm(x, w, torch.zeros_like(st)) == 0).all()
    wq, s = mb.quantize(w, mode="mxfp4")
    z = mb.grouped_qqmm(x, wq, s, st, mode="mxfp4")
    assert (z[17:] == 0).all() and (z[:17] != 0).any(1).all()
    ops.check_status()


@pytest.mark.parametrize("sizes,kept", (([30, 40, 5], [30, 20, 0]), ([-3, 20, 5], [0, 20, 5]), ([2 ** 40, 1, 1], [50, 0, 0]), ([50, -2 ** 40, 2 ** 62], [50, 0, 0])))
def test_sizes_that_do_not_fit_end_at_the_last_row_and_are_reported(sizes, kept):
    x, w, dy = randn(1, (50, 64), torch.bfloat16), randn(2, (3, 33, 64), torch.bfloat16), randn(3, (50, 33), torch.bfloat16)
    ops.check_status()
    st, ok = torch.tensor(sizes, device="cuda"), torch.tensor(kept, device="cuda")
    for f in (lambda s: mb.grouped_mm(x, w, s), lambda s: mb.grouped_mm_dw(dy, x, s)):
        y = f(st)
        with pytest.raises(ops.DeviceStatusError) as e:
            ops.check_status()
        assert e.value.code == 9
        assert torch.equal(y, f(ok))
        ops.check_status()


def test_empty_problems():
    bf = dict(dtype=torch.bfloat16, device="cuda")
    n = torch.zeros(2, dtype=torch.int64, device="cuda")
    assert mb.grouped_mm(torch.zeros(0, 8, **bf), torch.zeros(2, 5, 8, **bf), n).shape == (0, 5)
    assert (mb.grouped_mm(torch.zeros(3, 0, **bf), torch.zeros(2, 5, 0, **bf), n) == 0).all()
    assert mb.grouped_mm(torch.zeros(3, 8, **bf), torch.zeros(2, 0, 8, **bf), n).shape == (3, 0)
    assert (mb.grouped_mm(torch.ones(3, 8, **bf), torch.zeros(0, 5, 8, **bf), n[:0]) == 0).all()
    assert (mb.grouped_mm_dw(torch.zeros(0, 5, **bf), torch.zeros(0, 8, **bf), n) == 0).all()
    assert mb.grouped_mm_dw(torch.zeros(3, 5, **bf), torch.zeros(3, 0, **bf), n).shape == (2, 5, 0)
    ops.check_status()


def test_views_addresses_and_streams():
    flat = randn(1, (1 + 40 * 64,), torch.float16)
    w, st = randn(2, (2, 48, 64), torch.float16), torch.tensor([13, 27], device="cuda")
    x = flat[1:].reshape(40, 64)
    y = mb.grouped_mm(x.clone(), w, st)
    assert torch.equal(y, mb.grouped_mm(x, w, st))
    assert torch.equal(y, mb.grouped_mm(x.t().contiguous().t(), w.transpose(1, 2).contiguous().transpose(1, 2), st))
    assert torch.equal(y, mb.grouped_mm(x, w.transpose(1, 2).contiguous(), st, transpose=False))
    assert torch.equal(y, mb.grouped_mm(x, w, torch.stack((st, st), 1)[:, 0]))
    assert torch.equal(y, mb.grouped_mm(x, w, st.to(torch.int16)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mb.grouped_mm(x, w, st)
        graph = torch.cuda.CUDAGraph()
        n = st.clone()
        with torch.cuda.graph(graph, stream=side):
            z = mb.grouped_mm(x, w, n)
        for sizes in ((13, 27), (40, 0), (0, 21)):   # sizes change under a captured graph
            n.copy_(torch.tensor(sizes))
            graph.replay()
            side.synchronize()
            assert torch.equal(z, mb.grouped_mm(x, w, n))
    ops.check_status()


@pytest.mark.parametrize("transpose", (True, False))
@pytest.mark.parametrize("frozen", (None, "x", "w"))
def test_autograd(transpose, frozen):
    """Against the formulas, as views and through a broadcast cotangent, and against differences: the product is linear in x and in
    w, so a difference of any step is the derivative up to the roundings of the two results."""
    sizes, N, K = [7, 0, 30, 1], 40, 72
    T = sum(sizes)
    st = torch.tensor(sizes, device="cuda")
    x0, w0 = randn(1, (T, K), torch.bfloat16), randn(2, (4, N, K) if transpose else (4, K, N), torch.bfloat16)
    x, w = x0.clone().requires_grad_(frozen != "x"), w0.clone().requires_grad_(frozen != "w")
    y = grad.grouped_mm(x, w, st, transpose)
    assert torch.equal(y, mb.grouped_mm(x0, w0, st, transpose))
    dy = randn(3, (T, N), torch.bfloat16)
    y.backward(dy)
    if frozen != "x":
        assert torch.equal(x.grad, mb.grouped_mm(dy, w0, st, not transpose))
    else:
        assert x.grad is None
    if frozen != "w":
        assert torch.equal(w.grad, mb.grouped_mm_dw(dy, x0, st, transpose))
    else:
        assert w.grad is None
    D = plain.f64(dy)
    for arg, g, base in (("x", x.grad, x0), ("w", w.grad, w0)):
        if g is None:
            continue
        v = randn(4, base.shape, torch.bfloat16)
        up, down = (mb.grouped_mm(base + v, w0, st, transpose), mb.grouped_mm(base - v, w0, st, transpose)) if arg == "x" else \
                   (mb.grouped_mm(x0, base + v, st, transpose), mb.grouped_mm(x0, base - v, st, transpose))
        step = (plain.f64(base + v) - plain.f64(base - v)) / 2   # what was added in bf16
        a, b = (D * (plain.f64(up) - plain.f64(down)) / 2).sum(), (step * plain.f64(g)).sum()
        # half a unit of every result and of every element of the gradient, each at its largest
        room = 2.0 ** -9 * ((np.abs(D) * (np.abs(plain.f64(up)) + np.abs(plain.f64(down))) / 2).sum() + np.abs(step * plain.f64(g)).sum()) * 1.01
        assert abs(a - b) <= room, (a, b, room)
    # a cotangent that is broadcast (the sum's), and outputs used twice
    x, w = x0.clone().requires_grad_(), w0.clone().requires_grad_()
    y = grad.grouped_mm(x, w, st, transpose)
    (y.sum() + y.sum()).backward()
    ones = torch.full((T, N), 2.0, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(x.grad, mb.grouped_mm(ones, w0, st, not transpose)) and torch.equal(w.grad, mb.grouped_mm_dw(ones, x0, st, transpose))
    with torch.no_grad():
        assert not grad.grouped_mm(x, w, st, transpose).requires_grad


def test_autograd_of_other_inputs():
    """Views and odd addresses (the Python form), and of an activation that other operators made."""
    st = torch.tensor([5, 8], device="cuda")
    w = randn(1, (2, 24, 16), torch.bfloat16).requires_grad_()
    a = randn(2, (16, 13), torch.bfloat16).requires_grad_()
    y = grad.grouped_mm(a.t() * 2, w, st)
    dy = randn(3, (13, 24), torch.bfloat16)
    y.backward(dy.t().contiguous().t())
    x = (a.detach().t() * 2).contiguous()
    assert torch.equal(a.grad, (mb.grouped_mm(dy, w.detach(), st, False) * 2).t())
    assert torch.equal(w.grad, mb.grouped_mm_dw(dy, x, st))
    v = a.detach().t().requires_grad_()
    grad.grouped_mm(v, w, st).backward(dy)
    assert torch.equal(v.grad, mb.grouped_mm(dy, w.detach(), st, False))


def test_many_groups():
    """A table of more groups than a warp has lanes; the most that a call takes."""
    E, N, K = 4096, 8, 16
    sizes = (torch.arange(E) % 3).tolist()
    T = sum(sizes)
    x, w = randn(1, (T, K), torch.bfloat16), randn(2, (E, N, K), torch.bfloat16)
    st = torch.tensor(sizes, device="cuda")
    e = torch.repeat_interleave(torch.arange(E, device="cuda"), st)
    ref = torch.einsum("tk,tnk->tn", x.double(), w.double()[e])
    mass = torch.einsum("tk,tnk->tn", x.double().abs(), w.double()[e].abs())
    close(mb.grouped_mm(x, w, st), ref.cpu().numpy(), mass.cpu().numpy(), K, torch.bfloat16)
    with pytest.raises(RuntimeError, match="4096 groups"):
        mb.grouped_mm(x, randn(2, (E + 1, N, K), torch.bfloat16), torch.zeros(E + 1, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("mode", ("mxfp4", "nvfp4"))
def test_the_example_layer_learns_and_is_served_in_4_bits(mode):
    """Two 4-bit factors are off by about 0.13 of a product's norm (each value by 0.09 to 0.11 of its group's), two products in a row by
    about 0.2; wrong scales, rows or experts make it 1 and more."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "moe_layer.py")
    spec = importlib.util.spec_from_file_location("moe_layer", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    first, last, error = m.run(tokens=300, experts=6, width=192, hidden=320, steps=12, mode=mode)
    assert last < first and error < 0.4
    ops.check_status()
