"""dispatch_rows, combine_rows and their gradients against 64 bits."""
import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import grad

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def randn(seed, shape, dtype=torch.float32, std=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def routed(seed, T, E, top, off=0.0):
    """A routing of T tokens; a part `off` of the logits is -inf, so that some pairs have no expert."""
    logits = randn(seed, (T, E))
    logits[torch.rand((T, E), generator=torch.Generator("cuda").manual_seed(seed), device="cuda") < off] = float("-inf")
    return mb.route_experts(logits, top)


def near(got, ref, mass, terms):
    """fp32 sums of `terms` products: off by 2^-24 of the magnitudes' sum per term and product; then half a unit of the type."""
    t = torch.finfo(got.dtype)
    room = (terms + 1) * 2.0 ** -24 * mass
    assert ((got.double() - ref).abs() <= room + t.eps / 2 * (ref.abs() + room) + t.smallest_normal * t.eps).all()


def plain(r, x, y, w):
    """Rows by pair: x of the pair's token, y of its place (zeros where it has none)."""
    has = r.places >= 0
    yp = torch.where(has[..., None], y.double()[r.places.clamp_min(0).long()], 0.0)
    return has, yp


SHAPES = ((1, 1, 1), (1, 8, 2), (5, 4, 3), (67, 16, 6), (300, 60, 8), (9, 40, 32))
WIDTHS = (1, 7, 64, 1000, 2056, 4099)


@pytest.mark.parametrize("T,E,top", SHAPES)
@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype", tuple(DTYPES))
@pytest.mark.parametrize("off", (0.0, 0.5))
def test_both_directions_and_their_gradients(T, E, top, D, dtype, off):
    dt = DTYPES[dtype]
    r = routed(1, T, E, top, off)
    x, y = randn(2, (T, D), dt), randn(3, (T * top, D), dt)
    w = randn(4, (T, top))
    r = r._replace(weights=w)
    used = int(r.sizes.sum())
    y[used:] = float("nan")   # rows that belong to no pair are not read
    has, yp = plain(r, x, y, w)
    xs = mb.dispatch_rows(x, r)
    assert xs.shape == (T * top, D) and torch.equal(xs[:used], x[r.order[:used].long() // top]) and (xs[used:] == 0).all()
    out = mb.combine_rows(y, r)
    wd = torch.where(has, w.double(), 0.0)
    assert out.dtype == dt and out.shape == (T, D)
    near(out, torch.einsum("tj,tjd->td", wd, yp), torch.einsum("tj,tjd->td", wd.abs(), yp.abs()), top)
    near(mb.combine_rows(y, r, weighted=False), yp.sum(1), yp.abs().sum(1), top)
    dy = randn(5, (T, D), dt)
    dys, dw = mb.combine_rows_grad(dy, y, r)
    token, pair = r.order[:used].long() // top, r.order[:used].long()
    near(dys[:used], w.double().flatten()[pair][:, None] * dy.double()[token], torch.zeros((), device="cuda"), 0)
    assert (dys[used:] == 0).all()
    near(dw, torch.einsum("td,tjd->tj", dy.double(), yp), torch.einsum("td,tjd->tj", dy.double().abs(), yp.abs()), D)
    assert (dw[~has] == 0).all()
    only = mb.combine_rows_grad(dy, y, r, for_weights=False), mb.combine_rows_grad(dy, y, r, for_y=False)
    assert only[0][1] is None and only[1][0] is None and torch.equal(only[0][0], dys) and torch.equal(only[1][1], dw)


@pytest.mark.parametrize("dtype", tuple(DTYPES))
def test_autograd(dtype):
    """Against the calls' own gradients and, the sums being linear in every input, against differences."""
    dt, T, E, top, D = DTYPES[dtype], 40, 8, 3, 72
    r = routed(6, T, E, top, 0.3)
    x, y, w = randn(7, (T, D), dt).requires_grad_(), randn(8, (T * top, D), dt).requires_grad_(), randn(9, (T, top)).requires_grad_()
    r = r._replace(weights=w)
    xs, out = grad.dispatch_rows(x, r), grad.combine_rows(y, r)
    assert torch.equal(xs, mb.dispatch_rows(x, r)) and torch.equal(out, mb.combine_rows(y, r))
    dxs, dy = randn(10, xs.shape, dt), randn(11, out.shape, dt)
    dx, dys, dw = torch.autograd.grad((xs, out), (x, y, w), (dxs, dy))
    plain_r = r._replace(weights=w.detach())
    assert torch.equal(dx, mb.combine_rows(dxs, plain_r, weighted=False))
    assert all(torch.equal(a, b) for a, b in zip((dys, dw), mb.combine_rows_grad(dy, y.detach(), plain_r)))
    eps = torch.finfo(dt).eps
    for arg, base, g in (("y", y, dys), ("w", w, dw)):
        v = randn(12, base.shape, base.dtype)
        call = (lambda t: mb.combine_rows(t, plain_r)) if arg == "y" else (lambda t: mb.combine_rows(y.detach(), plain_r._replace(weights=t)))
        up, down = call((base + v).detach()).double(), call((base - v).detach()).double()
        step = ((base + v).detach().double() - (base - v).detach().double()) / 2
        a, b = (dy.double() * (up - down) / 2).sum(), (step * g.double()).sum()
        # half a unit of every result and gradient, and D + 2 half units of fp32 of every sum's terms
        terms = (dy.double().abs() * (up.abs() + down.abs()) / 2).sum() + (step * g.double()).abs().sum()
        mass = (dy.double().abs() * (up.abs() + down.abs() + 8 * y.detach().double().abs().max() * w.detach().double().abs().max() * top)).sum()
        assert (a - b).abs() <= (eps / 2 + 2.0 ** -23) * terms * 1.01 + (D + 2) * 2.0 ** -24 * mass
    # frozen inputs, a broadcast cotangent, outputs used twice, no gradient
    fy, = torch.autograd.grad(grad.combine_rows(y, plain_r), y, dy)
    fw, = torch.autograd.grad(grad.combine_rows(y.detach(), r), w, dy)
    assert torch.equal(fy, dys) and torch.equal(fw, dw)
    z = grad.dispatch_rows(x, r)
    (z.sum() + z.sum()).backward()
    assert torch.equal(x.grad, mb.combine_rows(torch.full_like(xs, 2.0), plain_r, weighted=False))
    with torch.no_grad():
        assert not grad.combine_rows(y, r).requires_grad and not grad.dispatch_rows(x, r).requires_grad
    g, = torch.autograd.grad(grad.combine_rows(y, r), y, dy.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_views_addresses_streams_and_graphs():
    T, top, D = 50, 4, 64
    r = routed(13, T, 8, top)
    flat = randn(14, (1 + T * D,), torch.bfloat16)
    x = flat[1:].reshape(T, D)
    xs = mb.dispatch_rows(x.clone(), r)
    assert torch.equal(mb.dispatch_rows(x, r), xs)
    assert torch.equal(mb.dispatch_rows(x.t().contiguous().t(), r), xs)
    lead = mb.route_experts(randn(13, (T, 8)).reshape(5, 10, 8), top)
    assert torch.equal(mb.dispatch_rows(x.reshape(5, 10, D), lead), xs)
    out = mb.combine_rows(xs, r)
    assert torch.equal(mb.combine_rows(xs, lead), out.reshape(5, 10, D))
    wide = torch.zeros((T * top, 2 * D), dtype=torch.bfloat16, device="cuda")
    wide[:, ::2] = xs
    assert torch.equal(mb.combine_rows(wide[:, ::2], r), out)
    assert torch.equal(mb.combine_rows(xs, r._replace(weights=r.weights.double())), out)
    # strided weights and plans
    both = torch.stack((r.weights, r.weights), -1)[..., 0]
    assert torch.equal(mb.combine_rows(xs, r._replace(weights=both, places=torch.stack((r.places, r.places), -1)[..., 0])), out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mb.combine_rows(mb.dispatch_rows(x, r), r)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            z = mb.combine_rows(mb.dispatch_rows(x, r), r)
        graph.replay()
    side.synchronize()
    assert torch.equal(z, out)


def test_infinities_and_nans_stay_in_their_token():
    T, top, D = 30, 2, 40
    r = routed(15, T, 6, top)
    y = randn(16, (T * top, D), torch.bfloat16)
    ref = mb.combine_rows(y, r)
    y[r.places[11, 1].long()] = float("nan")
    out = mb.combine_rows(y, r)
    assert torch.isnan(out[11]).all() and torch.equal(out[:11], ref[:11]) and torch.equal(out[12:], ref[12:])


def test_places_outside_the_rows_are_left_out():
    """Neither read nor written, whatever the table says."""
    T, top, D = 8, 2, 32
    x, y = randn(17, (T, D)), randn(18, (T * top, D))
    places = torch.arange(T * top, dtype=torch.int32, device="cuda").reshape(T, top)
    order = torch.arange(T * top, dtype=torch.int32, device="cuda")
    w = torch.ones((T, top), device="cuda")
    places[3, 0], places[4, 1] = T * top, -2 ** 31
    r = mb.Routing(w, None, None, places, order)
    keep = torch.ones((T, top, 1), device="cuda")
    keep[3, 0], keep[4, 1] = 0, 0
    assert torch.equal(mb.combine_rows(y, r), (y.reshape(T, top, D) * keep).sum(1))
    xs = mb.dispatch_rows(x, r).reshape(T, top, D)
    assert torch.equal(xs[:3], x[:3, None].expand(3, top, D)) and torch.equal(xs[3, 1], x[3])
    _, dw = mb.combine_rows_grad(x, y, r)
    assert dw[3, 0] == 0 and dw[4, 1] == 0


def test_empty():
    r = mb.route_experts(torch.zeros(0, 4, device="cuda"), 2)
    assert mb.dispatch_rows(torch.zeros(0, 8, device="cuda"), r).shape == (0, 8)
    assert mb.combine_rows(torch.zeros(0, 8, device="cuda"), r).shape == (0, 8)
    r = mb.route_experts(torch.zeros(3, 4, device="cuda"), 2)
    assert mb.dispatch_rows(torch.zeros(3, 0, device="cuda"), r).shape == (6, 0)
    assert mb.combine_rows(torch.zeros(6, 0, device="cuda"), r).shape == (3, 0)
    _, dw = mb.combine_rows_grad(torch.zeros(3, 0, device="cuda"), torch.zeros(6, 0, device="cuda"), r)
    assert (dw == 0).all()


def test_rows_far_into_memory():
    """Rows beyond 2^31 elements."""
    T, top, D = 70000, 8, 4096
    r = routed(19, T, 16, top)
    y = torch.zeros((T * top, D), dtype=torch.bfloat16, device="cuda")
    at = r.places[[0, T // 2, T - 1]].long()
    y[at.flatten()] = 1.0
    out = mb.combine_rows(y, r, weighted=False)
    assert (out[[0, T // 2, T - 1]] == top).all() and out.float().sum() == 3 * top * D
    del y
    x = torch.zeros((T, D), dtype=torch.bfloat16, device="cuda")
    x[T - 1] = 2.0
    xs = mb.dispatch_rows(x, r)
    assert (xs[r.places[T - 1].long()] == 2).all() and xs.float().sum() == 2.0 * top * D
