"""group_rows, add_adapters and its gradients against 64 bits."""
import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import grad, ops

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def randn(seed, shape, dtype=torch.float32, std=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def problem(seed, ids, L, r, N, K, dt):
    T = ids.numel()
    return (randn(seed, (T, N), dt), randn(seed + 1, (T, K), dt), randn(seed + 2, (L, r, K), dt, K ** -0.5), randn(seed + 3, (L, N, r), dt, r ** -0.5),
            randn(seed + 4, (L,)).abs() + 0.5)


def exact(ids, y, x, a, b, scales, dy=None):
    """-> out and the magnitudes of its terms; with dy: dx, da, db and theirs."""
    y, x, a, b = (t.detach().double() for t in (y, x, a, b))
    c = torch.ones(a.shape[0], dtype=torch.float64, device="cuda") if scales is None else scales.double()
    out, mass = y.clone(), torch.zeros_like(y)
    if dy is not None:
        dy = dy.double()
        dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
        mx, ma, mb_ = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for l in range(a.shape[0]):
        at = (ids == l).nonzero()[:, 0]
        h, hm = x[at] @ a[l].T, x[at].abs() @ a[l].abs().T
        out[at] += c[l] * h @ b[l].T
        mass[at] = c[l] * hm @ b[l].abs().T
        if dy is not None:
            g, gm = c[l] * dy[at] @ b[l], c[l] * dy[at].abs() @ b[l].abs()
            dx[at], mx[at] = g @ a[l], gm @ a[l].abs()
            da[l], ma[l] = g.T @ x[at], gm.T @ x[at].abs()
            db[l], mb_[l] = c[l] * dy[at].T @ h, c[l] * dy[at].abs().T @ hm
    return (out, mass) if dy is None else ((dx, mx), (da, ma), (db, mb_))


def near(got, ref, mass, terms):
    """fp32 sums of `terms` terms in any order, truncated at each: 2^-23 of the magnitudes' sum each; the inner product as two bf16
    numbers and (f16) the product of two low parts left out: 2^-17 + 2^-16; then half a unit of the type."""
    t = torch.finfo(got.dtype)
    room = (terms * 2.0 ** -23 + 3 * 2.0 ** -17) * mass
    bad = (got.double() - ref).abs() - (room + t.eps / 2 * (ref.abs() + room) + 2.0 ** -23 * ref.abs() + t.smallest_normal * t.eps)
    assert (bad <= 0).all(), float(bad.max())


def ids_of(name):
    g = torch.Generator().manual_seed(5)
    return {"one": torch.tensor([0]), "none": torch.tensor([-1]), "own": torch.arange(7), "all none": torch.full((70,), -1),
            "mixed": torch.randint(-1, 5, (200,), generator=g), "runs": torch.tensor([2] * 65 + [-1] * 3 + [0] * 16 + [4] * 130 + [2] * 20),
            "long": torch.tensor([1] * 700 + [3] * 5), "outside": torch.tensor([0, 7, -9, 3, 2 ** 31 - 1, 1])}[name].cuda()


@pytest.mark.parametrize("name,L", (("one", 1), ("one", 3), ("none", 2), ("own", 7), ("all none", 2), ("mixed", 5), ("runs", 5), ("long", 4), ("outside", 4)))
@pytest.mark.parametrize("r,N,K,dtype,scaled", ((16, 256, 512, "bf16", True), (16, 264, 200, "f16", False), (8, 100, 130, "bf16", False), (1, 33, 17, "f16", True),
                                                (64, 520, 1000, "bf16", True), (20, 256, 136, "f16", True), (33, 72, 301, "bf16", True),
                                                (130, 296, 264, "f16", True), (6, 64, 2048, "bf16", False)))
def test_adapters_and_their_gradients(name, L, r, N, K, dtype, scaled):
    """Rows of one, no and many adapters, tiles with a row and full ones; ranks and widths that end inside every piece."""
    ids, dt = ids_of(name), DTYPES[dtype]
    y, x, a, b, scales = problem(1, ids, L, r, N, K, dt)
    scales = scales if scaled else None
    T = ids.numel()
    groups = mb.group_rows(ids, L)
    inside = (ids >= 0) & (ids < L)
    want = torch.where(inside, ids, L)
    order = want.argsort(stable=True)
    n = int(inside.sum())
    assert torch.equal(groups.order.long(), torch.where(torch.arange(T, device="cuda") < n, order, -1 - order))
    assert torch.equal(groups.sizes.long(), torch.bincount(want, minlength=L + 1)[:L])
    assert torch.equal(groups.starts.long(), torch.bincount(want, minlength=L + 1).cumsum(0) - torch.bincount(want, minlength=L + 1))
    out = mb.add_adapters(y, x, a, b, groups, scales)
    assert out.dtype == dt and torch.equal(out[~inside], y[~inside])
    near(out, *exact(ids, y, x, a, b, scales), K + r)
    assert torch.equal(out, mb.add_adapters(y, x, a, b, groups, scales))
    place = y.clone()
    assert mb.add_adapters(place, x, a, b, groups, scales, out=place) is place and torch.equal(place, out)
    dy = randn(9, (T, N), dt)
    leaves = [t.clone().requires_grad_() for t in (y, x, a, b)]
    z = grad.add_adapters(*leaves, groups, scales)
    assert torch.equal(z, out)
    d_y, *got = torch.autograd.grad(z, leaves, dy)
    assert torch.equal(d_y, dy)
    for g, (ref, mass), terms in zip(got, exact(ids, y, x, a, b, scales, dy), (N + r, T + N, T + K)):
        near(g, ref, mass, terms)
    assert (got[0][~inside] == 0).all()
    for l in range(L):
        if int(groups.sizes[l]) == 0:
            assert (got[1][l] == 0).all() and (got[2][l] == 0).all()


@pytest.mark.parametrize("T,L,r,N,K", ((1, 2, 16, 14336, 4096), (300, 3, 16, 4096, 8192), (1100, 40, 32, 1024, 4096), (5000, 2, 64, 512, 256)))
def test_parts_of_long_sums(T, L, r, N, K):
    """Long dimensions and many rows, cut over blocks, in every direction; the same bits every time."""
    ids = torch.randint(-1, L, (T,), generator=torch.Generator().manual_seed(2)).cuda()
    y, x, a, b, scales = problem(3, ids, L, r, N, K, torch.bfloat16)
    groups = mb.group_rows(ids.int(), L)
    out, h = ops._add_adapters(y, x, a, b, groups, scales)
    near(out, *exact(ids, y, x, a, b, scales), K + r)
    dy = randn(9, (T, N), torch.bfloat16)
    got = mb.add_adapters_grad(dy, x, a, b, groups, h, scales)
    for g, (ref, mass), terms in zip(got, exact(ids, y, x, a, b, scales, dy), (N + r, T + N, T + K)):
        near(g, ref, mass, terms)
    for _ in range(3):
        assert torch.equal(out, mb.add_adapters(y, x, a, b, groups, scales))
        assert all(torch.equal(p, q) for p, q in zip(got, mb.add_adapters_grad(dy, x, a, b, groups, h, scales)))
    for i, wanted in enumerate(((True, False, False), (False, True, False), (False, False, True))):
        some = mb.add_adapters_grad(dy, x, a, b, groups, h, scales, *wanted)
        assert torch.equal(some[i], got[i]) and sum(t is not None for t in some) == 1


@pytest.mark.parametrize("T,n", ((1, 0), (5, 1), (31, 3), (4096, 4096), (4097, 600), (100000, 1000), (300001, 70)))
@pytest.mark.parametrize("kind", (torch.int32, torch.int64, torch.int16))
def test_group_rows(T, n, kind):
    """One block and many, more groups than a warp has lanes, rows in uneven numbers."""
    g = torch.Generator().manual_seed(T)
    ids = (torch.randn(T, generator=g).abs() * n / 2).long() - 1
    ids = ids.clamp_max(2 ** 15 - 1).to(kind).cuda()
    r = mb.group_rows(ids, n)
    inside = (ids >= 0) & (ids < n)
    want = torch.where(inside, ids.long(), n)
    order, sizes = want.argsort(stable=True), torch.bincount(want, minlength=n + 1)
    have = int(inside.sum())
    assert torch.equal(r.order.long(), torch.where(torch.arange(T, device="cuda") < have, order, -1 - order))
    assert torch.equal(r.sizes.long(), sizes[:n]) and torch.equal(r.starts.long(), sizes.cumsum(0) - sizes)
    # every place is in one tile, of its group
    tiles = r.tiles.cpu().tolist()
    seen = torch.zeros(T, dtype=torch.int64)
    group_at = torch.repeat_interleave(torch.arange(n + 1), sizes.cpu())
    for l, first, rows, _ in tiles:
        assert 0 <= rows <= 64
        if rows:
            seen[first:first + rows] += 1
            assert (group_at[first:first + rows] == (l if l >= 0 else n)).all()
    assert (seen == 1).all()


def test_infinities_and_nans_stay_in_their_row_and_adapter():
    ids = torch.tensor([0] * 20 + [1] * 30 + [-1] * 4 + [2] * 10, device="cuda")
    y, x, a, b, s = problem(5, ids, 3, 16, 128, 256, torch.bfloat16)
    groups = mb.group_rows(ids, 3)
    dy = randn(9, y.shape, torch.bfloat16)
    ref, h = ops._add_adapters(y, x, a, b, groups, s)
    grads = mb.add_adapters_grad(dy, x, a, b, groups, h, s)
    for bad in (float("nan"), float("inf")):
        x2, a2, b2, dy2 = x.clone(), a.clone(), b.clone(), dy.clone()
        x2[20:50], a2[1], b2[1], dy2[20:50] = bad, bad, bad, bad
        out, h2 = ops._add_adapters(y, x2, a2, b2, groups, s)
        assert torch.equal(out[:20], ref[:20]) and torch.equal(out[50:], ref[50:]) and not torch.isfinite(out[20:50]).any()
        dx, da, db = mb.add_adapters_grad(dy2, x2, a2, b2, groups, h2, s)
        for got, want, own in ((dx, grads[0], slice(20, 50)), (da, grads[1], slice(1, 2)), (db, grads[2], slice(1, 2))):
            assert not torch.isfinite(got[own]).any()
            got[own], want = 0, want.clone()
            want[own] = 0
            assert torch.equal(got, want)
    x2 = x.clone()
    x2[5, 3] = float("inf")   # one infinity: every rank's is one, and their sum an infinity or (of both signs) a NaN
    out = mb.add_adapters(y, x2, a, b, groups, s)
    assert torch.equal(out[:5], ref[:5]) and torch.equal(out[6:], ref[6:]) and not torch.isfinite(out[5]).any()
    one = torch.zeros_like(a)
    one[:, 0] = a[:, 0]
    b1 = torch.zeros_like(b)
    b1[:, :, 0] = b[:, :, 0]
    out = mb.add_adapters(y, x, one, b1, groups, torch.full_like(s, float("inf")))
    h = x[0].double() @ a[0, 0].double()
    assert torch.isfinite(h)   # 0 times infinity in the other ranks
    assert not torch.isfinite(out[0]).any() and torch.equal(out[50:54], y[50:54])


@pytest.mark.parametrize("dtype", tuple(DTYPES))
def test_inner_products_beyond_the_type(dtype):
    """a x far above and below what float16 holds, the result inside it."""
    dt, N, K, r = DTYPES[dtype], 64, 64, 4
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    y, x, a, b, _ = problem(7, ids, 1, r, N, K, dt)
    groups = mb.group_rows(ids, 1)
    for size, c in ((2.0 ** 9, 2.0 ** -18), (2.0 ** -9, 2.0 ** 18)):
        x2, a2, s = (x.double() * size).to(dt), (a.double() * size).to(dt), torch.tensor([c], device="cuda")
        near(mb.add_adapters(y, x2, a2, b, groups, s), *exact(ids, y, x2, a2, b, s), K + r)


def test_views_addresses_types_and_streams():
    ids = torch.tensor([0, 1, 1, -1, 0] * 8, device="cuda")
    y, x, a, b, s = problem(8, ids, 2, 16, 96, 128, torch.float16)
    groups = mb.group_rows(ids, 2)
    ref = mb.add_adapters(y, x, a, b, groups, s)
    off = lambda t: torch.cat((t.new_zeros(1), t.flatten()))[1:].reshape(t.shape)   # not on a 16-byte boundary
    turned = lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)
    for f in (off, turned):
        for i in range(4):
            args = [y, x, a, b]
            args[i] = f(args[i])
            assert torch.equal(mb.add_adapters(*args, groups, s), ref)
    assert torch.equal(mb.add_adapters(y.reshape(5, 8, 96), x.reshape(5, 8, 128), a, b, groups, s).reshape(40, 96), ref)
    assert torch.equal(mb.add_adapters(y, x, a, b, groups, s.double()), ref)
    out = torch.empty_like(y)
    assert mb.add_adapters(y, x, a, b, groups, s, out=out) is out and torch.equal(out, ref)
    assert torch.equal(mb.add_adapters(y[0], x[0], a, b, mb.group_rows(ids[0], 2), s), ref[0])
    with pytest.raises(ValueError):
        mb.add_adapters(y, x, a, b, groups, s, out=torch.empty((40, 192), dtype=torch.float16, device="cuda")[:, ::2])
    both = torch.empty((41, 96), dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        mb.add_adapters(both[1:], x, a, b, groups, s, out=both[:40])
    square = mb.add_adapters(x, x, a, randn(3, (2, 128, 16), torch.float16), groups, s)   # y and x the same
    assert square.shape == x.shape
    with pytest.raises(ValueError):
        mb.add_adapters(x, x, a, randn(3, (2, 128, 16), torch.float16), groups, s, out=x)
    with pytest.raises(ValueError):
        mb.add_adapters(y, x, a, b, mb.group_rows(ids[:-1], 2), s)
    with pytest.raises(ValueError):
        mb.add_adapters(y, x, a, b, mb.group_rows(ids, 3), s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mb.add_adapters(y, x, a, b, groups, s)
        graph, n = torch.cuda.CUDAGraph(), ids.clone()
        with torch.cuda.graph(graph, stream=side):
            z = mb.add_adapters(y, x, a, b, mb.group_rows(n, 2), s)
        for other in (ids, ids.flip(0), torch.full_like(ids, -1), torch.ones_like(ids)):   # requests change under a captured graph
            n.copy_(other)
            graph.replay()
            side.synchronize()
            assert torch.equal(z, mb.add_adapters(y, x, a, b, mb.group_rows(other, 2), s))


def test_tables_that_do_not_fit_are_not_followed():
    """Entries outside the operands are left out: nothing is read or written there."""
    ids = torch.tensor([0, 1, 1, 0], device="cuda")
    y, x, a, b, s = problem(10, ids, 2, 8, 64, 64, torch.bfloat16)
    groups = mb.group_rows(ids, 2)
    bad = groups.tiles.clone()
    bad[0] = torch.tensor([9, 0, 2, 4])
    bad[1] = torch.tensor([0, 3, 60, 4])
    out = torch.zeros_like(y)
    mb.add_adapters(y, x, a, b, groups._replace(tiles=bad), s, out=out)
    assert (out == 0).all()
    far = groups.order.clone()
    far[2] = 1000
    mb.add_adapters(y, x, a, b, groups._replace(order=far), s)
    torch.cuda.synchronize()


def test_empty():
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")
    none = mb.group_rows(torch.zeros(0, dtype=torch.int64, device="cuda"), 3)
    assert mb.add_adapters(z(0, 8), z(0, 4), z(3, 2, 4), z(3, 8, 2), none).shape == (0, 8)
    ids = torch.tensor([0, 1], device="cuda")
    one = torch.ones((2, 8), dtype=torch.bfloat16, device="cuda")
    g = mb.group_rows(ids, 0)
    assert torch.equal(mb.add_adapters(one, z(2, 4), z(0, 2, 4), z(0, 8, 2), g), one)
    g = mb.group_rows(ids, 3)
    assert torch.equal(mb.add_adapters(one, z(2, 4), z(3, 0, 4), z(3, 8, 0), g), one)
    assert torch.equal(mb.add_adapters(one, z(2, 0), z(3, 2, 0), z(3, 8, 2), g), one)
    assert mb.add_adapters(z(2, 0), z(2, 4), z(3, 2, 4), z(3, 0, 2), g).shape == (2, 0)
    a, b = z(3, 2, 4).requires_grad_(), z(3, 0, 2).requires_grad_()
    da, db = torch.autograd.grad(grad.add_adapters(z(2, 0), z(2, 4), a, b, g).sum(), (a, b))
    assert (da == 0).all() and db.shape == b.shape


def test_autograd_modes():
    """Frozen inputs, a broadcast cotangent, no gradient, second order (refused), a backward pass captured while an eager graph of the same
    leaves lives, and differences: the sum is linear in every input."""
    ids = torch.tensor([0, 1, -1, 1] * 10, device="cuda")
    y, x, a, b, s = problem(11, ids, 2, 8, 40, 72, torch.bfloat16)
    groups = mb.group_rows(ids, 2)
    dy = randn(9, y.shape, torch.bfloat16)
    _, h = ops._add_adapters(y, x, a, b, groups, s)
    ref = (dy, *mb.add_adapters_grad(dy, x, a, b, groups, h, s))
    for i in range(4):
        args = [y, x, a, b]
        args[i] = args[i].clone().requires_grad_()
        g, = torch.autograd.grad(grad.add_adapters(*args, groups, s), args[i], dy)
        assert torch.equal(g, ref[i])
    leaves = [t.clone().requires_grad_() for t in (y, x, a, b)]
    with torch.no_grad():
        assert not grad.add_adapters(*leaves, groups, s).requires_grad
    grad.add_adapters(*leaves, groups, s).sum().backward()
    ones = torch.ones_like(dy)
    assert all(torch.equal(t.grad, g) for t, g in zip(leaves, (ones, *mb.add_adapters_grad(ones, x, a, b, groups, h, s))))
    g, = torch.autograd.grad(grad.add_adapters(*leaves, groups, s), leaves[1:2], dy, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
    D = dy.double()
    for i in (1, 2, 3):
        args = [y, x, a, b]
        v = randn(12, args[i].shape, torch.bfloat16, float(args[i].float().std()))
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + v, args[i] - v
        step = (up[i].double() - down[i].double()) / 2
        p, q = (mb.add_adapters(*t, groups, s).double() for t in (up, down))
        one, two = (D * (p - q) / 2).sum(), (step * ref[i].double()).sum()
        # half a unit of every result and gradient, and the inner products' and sums' errors (2^-14 of the terms, of which the results hold
        # a tenth at least)
        room = (2.0 ** -9 + 10 * 2.0 ** -14) * ((D.abs() * (p.abs() + q.abs()) / 2).sum() + (step * ref[i].double()).abs().sum()) * 1.01
        assert (one - two).abs() <= room
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        fresh = [t.detach().clone().requires_grad_() for t in leaves]
        torch.autograd.grad(grad.add_adapters(*fresh, groups, s), fresh, dy)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            got = torch.autograd.grad(grad.add_adapters(*fresh, groups, s), fresh, dy)
        graph.replay()
    st.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, ref))


def test_beside_a_quantized_projection():
    """As it is used: one quantized projection for the batch, the adapters in place on top."""
    ids = torch.tensor([1, 0, -1, 1, 2], device="cuda")
    y, x, a, b, s = problem(13, ids, 3, 16, 256, 512, torch.bfloat16)
    w = mb.quantize(randn(14, (256, 512), torch.bfloat16, 0.05))
    y = mb.quantized_matmul(x, *w)
    groups = mb.group_rows(ids, 3)
    out = mb.add_adapters(y.clone(), x, a, b, groups, s)
    near(out, *exact(ids, y, x, a, b, s), 512 + 16)


def test_sums_in_place_and_autograd():
    """What is overwritten is noticed by a graph that has kept it; a sum in place of what is part of a graph is refused."""
    ids = torch.tensor([1, 0, -1, 1], device="cuda")
    y, x, a, b, s = problem(15, ids, 2, 8, 64, 72, torch.bfloat16)
    groups = mb.group_rows(ids, 2)
    ref = mb.add_adapters(y, x, a, b, groups, s)
    for into in (lambda kept: kept, lambda kept: y):   # in place; another tensor's sum
        for scales in (s, s.double()):
            kept, w = y.clone(), torch.ones_like(y).requires_grad_()
            z = kept * w
            mb.add_adapters(into(kept), x, a, b, groups, scales, out=kept)
            assert torch.equal(kept, ref)
            with pytest.raises(RuntimeError):
                z.sum().backward()
    leaf = y.clone().requires_grad_()
    for t in (leaf, leaf * 2):
        with pytest.raises(ValueError):
            mb.add_adapters(t, x, a, b, groups, s, out=t)
        with pytest.raises(ValueError):
            mb.add_adapters(y, x, a, b, groups, s, out=t)
    assert torch.equal(leaf, y)
    with torch.no_grad():
        assert torch.equal(mb.add_adapters(leaf, x, a, b, groups, s, out=leaf), ref)
    with torch.inference_mode():
        t = y.clone()
        assert torch.equal(mb.add_adapters(t, x, a, b, groups, s, out=t), ref)


@pytest.mark.parametrize("T,N,K,r,dtype", ((32000, 1032, 72, 33, "f16"), (16000, 1030, 64, 66, "f16"), (700, 38200, 64, 33, "f16"), (9000, 8200, 64, 4, "bf16")))
@pytest.mark.parametrize("last", (0.0, 0.9))
def test_many_tiles(T, N, K, r, dtype, last):
    """Many tiles per block of the second product, and columns for more blocks than there is room for; with some rows or most of them without an adapter."""
    g = torch.Generator().manual_seed(21)
    ids = torch.randint(-1, 3, (T,), generator=g)
    ids[torch.rand(T, generator=g) < last] = -1
    ids = ids.cuda()
    y, x, a, b, s = problem(22, ids, 4, r, N, K, DTYPES[dtype])
    groups = mb.group_rows(ids, 4)
    out = mb.add_adapters(y, x, a, b, groups, s)
    near(out, *exact(ids, y, x, a, b, s), K + r)
    y2 = y.clone()
    mb.add_adapters(y2, x, a, b, groups, s, out=y2)
    assert torch.equal(y2, out)
    _, h = ops._add_adapters(y, x, a, b, groups, s)
    dx, _, _ = mb.add_adapters_grad(y, x, a, b, groups, h, s, True, False, False)
    assert (dx[ids < 0] == 0).all()
