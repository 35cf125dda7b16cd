"""route_experts and its gradient against 64 bits: the same experts always, weights up to their roundings."""
import numpy as np
import pytest
import torch

import mlx_b200 as mb
import routing_plain as plain
from mlx_b200 import grad

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF = float("inf")


def randn(seed, shape, dtype=torch.float32, std=1.5):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def f64(t):
    return t.detach().double().cpu().numpy()


def close(w, ref, logits):
    """Half units (2^-24 of the weight) that are lost: of both exponentials the argument's rounding, at most the range R of the row's
    logits, and 4 of exp itself; 37 of a sum of up to 32 terms per lane over 32 lanes; sigmoid's sum, divisions, products: 8."""
    finite = np.where(np.isfinite(logits), logits, 0.0)
    span = (finite.max(-1) - finite.min(-1))[:, None] + np.abs(finite).max(-1)[:, None]
    assert (np.abs(f64(w) - ref) <= np.abs(ref) * (2 * span + 53) * 2.0 ** -24 + 2.0 ** -140).all()


def check(logits, top, bias=None, **kw):
    r = mb.route_experts(logits, top, bias=bias, **kw)
    l = f64(logits)
    ref = plain.route(l, top, bias=None if bias is None else f64(bias), **kw)
    for got, want, name in zip(r[1:], ref[1:], r._fields[1:]):
        assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), want), name
    assert r.weights.dtype == torch.float32
    close(r.weights, ref[0], l)
    return r


SHAPES = ((1, 1, 1, 1, 1), (1, 8, 2, 1, 1), (5, 4, 4, 2, 1 + 1), (3, 33, 5, 1, 1), (64, 64, 8, 4, 2), (65, 60, 4, 6, 2), (130, 256, 8, 8, 4), (260, 96, 32, 1, 1),
          (33, 1000, 7, 10, 3), (129, 1024, 32, 32, 5), (700, 160, 6, 8, 3))


@pytest.mark.parametrize("T,E,top,groups,top_groups", SHAPES)
@pytest.mark.parametrize("scoring", ("softmax", "sigmoid"))
@pytest.mark.parametrize("biased", (False, True))
@pytest.mark.parametrize("best,dtype,renormalize,scale", ((1, "f32", True, 1.0), (2, "bf16", False, 2.5), (1, "f16", False, 1.0), (2, "f32", True, 0.5)))
def test_against_64_bits(T, E, top, groups, top_groups, scoring, biased, best, dtype, renormalize, scale):
    """One block and several, every number of experts per lane, groups of one expert and more, every choice of arguments."""
    bias = randn(2, (E,), std=0.2) if biased else None
    check(randn(1, (T, E), DTYPES[dtype]), top, bias, scoring=scoring, groups=groups, top_groups=top_groups, group_best=best,
          renormalize=renormalize, scale=scale)


@pytest.mark.parametrize("T", (7, 300))
@pytest.mark.parametrize("bias", (None, "zeros", "few"))
def test_ties_go_to_the_lowest_index(T, bias):
    E = 96
    logits = torch.randint(-2, 3, (T, E), generator=torch.Generator().manual_seed(1)).float().cuda()
    logits[0] = 0.0
    logits[1, ::2] = -0.0   # equal to 0
    b = None if bias is None else torch.zeros(E, device="cuda")
    if bias == "few":
        b[::3] = 0.25
    for kw in (dict(), dict(groups=8, top_groups=3)):
        check(logits, 9, b, scoring="sigmoid", **kw)
        check(logits, 9, b, scoring="softmax", renormalize=True, **kw)


@pytest.mark.parametrize("scoring", ("softmax", "sigmoid"))
@pytest.mark.parametrize("groups,best", ((1, 1), (8, 1), (8, 2)))
def test_keys_that_32_bits_cannot_tell_apart(scoring, groups, best):
    """Every bias is a constant less the first token's score, rounded: all its keys are within a rounding of each other."""
    E = 256
    logits = randn(3, (40, E))
    s = torch.softmax(logits.double(), -1) if scoring == "softmax" else torch.sigmoid(logits.double())
    for t in (0, 5):
        check(logits, 8, (0.5 - s[t]).float(), scoring=scoring, groups=groups, top_groups=max(1, groups // 2), group_best=best)


def test_group_ranks_that_32_bits_cannot_tell_apart():
    """Without a bias, groups whose two best scores have sums next to each other; the experts then go by their logits."""
    G, E = 16, 64
    a = torch.linspace(-1.0, 1.0, G, dtype=torch.float64)
    b = torch.logit(1.2 - torch.sigmoid(a))   # sigmoid(a) + sigmoid(b) = 1.2
    logits = torch.full((1, G, E // G), -9.0, dtype=torch.float64)
    logits[0, :, 1], logits[0, :, 3] = a, b
    logits = logits.reshape(1, E).float().cuda().repeat(3, 1)
    logits[1:] += 0.001
    check(logits, 6, scoring="sigmoid", groups=G, top_groups=5, group_best=2)


@pytest.mark.parametrize("scoring", ("softmax", "sigmoid"))
@pytest.mark.parametrize("renormalize", (False, True))
@pytest.mark.parametrize("dtype", tuple(DTYPES))
@pytest.mark.parametrize("T", (10, 200))
def test_experts_that_are_off(scoring, renormalize, dtype, T):
    """-inf among the logits: never taken, even with the largest bias; rows with fewer than `top` left, and with none."""
    E, top = 40, 6
    logits = randn(4, (T, E), DTYPES[dtype])
    logits[0] = -INF
    logits[1, 3:] = -INF
    logits[2, :34] = -INF
    logits[3, ::2] = -INF
    logits[-1] = -INF
    for bias in (None, randn(5, (E,), std=3.0)):
        for kw in (dict(), dict(groups=4, top_groups=2), dict(groups=4, top_groups=2, group_best=2)):
            r = check(logits, top, bias, scoring=scoring, renormalize=renormalize, **kw)
            assert (r.experts[0] == -1).all() and (r.weights[0] == 0).all() and (r.places[-1] == -1).all()
    bias = torch.zeros(E, device="cuda")
    bias[:30] = -INF
    check(logits, top, bias, scoring=scoring, renormalize=renormalize)
    all_off = mb.route_experts(torch.full((T, E), -INF, device="cuda"), top, scoring)
    assert (all_off.sizes == 0).all() and torch.equal(all_off.order, -1 - torch.arange(T * top, device="cuda", dtype=torch.int32))


@pytest.mark.parametrize("dtype", tuple(DTYPES))
def test_masks_of_the_lowest_value_and_far_logits(dtype):
    """The type's lowest number is a number: such an expert comes last but is there; scores that underflow still have ratios."""
    dt, E = DTYPES[dtype], 24
    logits = randn(6, (20, E), dt)
    logits[:, 5:] = torch.finfo(dt).min
    for scoring in ("softmax", "sigmoid"):
        check(logits, 8, scoring=scoring)
    r = mb.route_experts(logits, 8, "softmax", renormalize=True)
    assert (r.weights[:, 5:] == 0).all() and torch.allclose(r.weights.sum(-1), torch.ones(20, device="cuda"))
    far = randn(7, (20, E), dt) - 200.0
    for scoring in ("softmax", "sigmoid"):
        check(far, 4, scoring=scoring, renormalize=True)


def test_nan_and_infinity():
    logits = randn(8, (6, 33))
    logits[0, 7] = float("nan")
    logits[1, [4, 30]] = float("nan")
    logits[2] = float("nan")
    logits[3, 9] = INF
    clean = mb.route_experts(logits[4:], 4)
    for scoring in ("softmax", "sigmoid"):
        for bias in (None, torch.zeros(33, device="cuda")):
            r = mb.route_experts(logits, 4, scoring, bias)
            e = r.experts.cpu()
            if scoring == "softmax" and bias is not None:   # a NaN makes every score of its row one: equal keys
                assert e[:3].tolist() == [[0, 1, 2, 3]] * 3
            else:
                assert e[0, 0] == 7 and e[1, :2].tolist() == [4, 30] and e[2].tolist() == [0, 1, 2, 3]
            assert sorted(r.order.tolist()) == list(range(24)) and ((e >= 0) & (e < 33)).all()
            if bias is None:
                assert e[3, 0] == 9
            if scoring == "sigmoid":
                assert r.weights[3][r.experts[3] == 9] == 1 and torch.isnan(r.weights[0, 0]) and not torch.isnan(r.weights[0, 1:]).any()
            else:
                assert torch.isnan(r.weights[:3]).all()
    assert torch.equal(mb.route_experts(logits, 4).weights[4:], clean.weights)


def test_empty_strided_and_leading_dimensions():
    logits = randn(9, (6, 5, 16))
    r = mb.route_experts(logits, 3)
    flat = mb.route_experts(logits.reshape(30, 16), 3)
    assert r.weights.shape == r.experts.shape == r.places.shape == (6, 5, 3) and torch.equal(r.order, flat.order)
    assert torch.equal(r.experts.reshape(30, 3), flat.experts)
    wide = randn(10, (30, 40))
    wide[:, 3:35:2] = logits.reshape(30, 16)
    for a, b in zip(mb.route_experts(wide[:, 3:35:2], 3), flat):
        assert torch.equal(a, b)
    one = mb.route_experts(logits[0, 0], 3)
    assert one.weights.shape == (3,) and one.order.shape == (3,)
    none = mb.route_experts(logits[:0], 3)
    assert none.weights.shape == (0, 5, 3) and none.order.shape == (0,) and (none.sizes == 0).all()
    b = randn(11, (32,), torch.float64)[::2]
    assert torch.equal(mb.route_experts(logits, 3, bias=b).experts, mb.route_experts(logits, 3, bias=b.float().contiguous()).experts)


def test_many_tokens():
    """Several tokens per warp and all blocks, experts in uneven numbers; the same every time."""
    T, E, top = 50001, 60, 4
    logits = randn(12, (T, E), torch.bfloat16)
    logits[:, 17] += 8.0   # nearly everyone's first
    logits[:, 3] = -INF    # nobody's
    r = mb.route_experts(logits, top, renormalize=True)
    l = logits.double()
    want = l.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(r.experts.long(), want)
    order = want.flatten().argsort(stable=True)
    assert torch.equal(r.order.long(), order) and torch.equal(r.sizes.long(), torch.bincount(want.flatten(), minlength=E))
    assert torch.equal(r.places.flatten().long()[order], torch.arange(T * top, device="cuda"))
    assert all(torch.equal(a, b) for _ in range(3) for a, b in zip(r, mb.route_experts(logits, top, renormalize=True)))


def test_streams_and_graphs():
    """Two captured graphs that are replayed at the same time, and eager calls between them."""
    a, b = randn(13, (500, 64)), randn(14, (700, 64))
    ra, rb = mb.route_experts(a, 6), mb.route_experts(b, 6)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for st, x in zip(side, (a, b)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mb.route_experts(x, 6))
        graphs.append(g)
    for _ in range(10):
        for st, g in zip(side, graphs):
            with torch.cuda.stream(st):
                g.replay()
        c = mb.route_experts(a, 6)
        torch.cuda.synchronize()
        for got, want in ((outs[0], ra), (outs[1], rb), (c, ra)):
            assert all(torch.equal(p, q) for p, q in zip(got, want))
    a.copy_(randn(15, (500, 64)))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs[0], mb.route_experts(a, 6)))


# ---------------------------------------------------------------------------------------------------- gradient
def exact_gradient(logits, experts, dw, scoring, renormalize, scale):
    """From the definition, differentiated in 64 bits; pairs without an expert have no weight."""
    l = logits.detach().double().requires_grad_()
    has = experts >= 0
    logp = torch.log_softmax(l, -1) if scoring == "softmax" else torch.nn.functional.logsigmoid(l)
    chosen = torch.where(has, logp.gather(1, experts.clamp_min(0).long()), -INF)
    w = (torch.softmax(chosen, -1) if renormalize else chosen.exp()) * scale
    g, = torch.autograd.grad(w, l, torch.where(has, dw.double(), 0.0))
    return g


@pytest.mark.parametrize("T,E,top", ((1, 1, 1), (9, 8, 2), (70, 60, 4), (33, 256, 8), (65, 1000, 32)))
@pytest.mark.parametrize("scoring", ("softmax", "sigmoid"))
@pytest.mark.parametrize("renormalize", (False, True))
@pytest.mark.parametrize("dtype", tuple(DTYPES))
def test_gradient(T, E, top, scoring, renormalize, dtype):
    dt, scale = DTYPES[dtype], 1.5
    logits = randn(16, (T, E), dt).requires_grad_()
    if E > 30:
        with torch.no_grad():
            logits[0, ::3] = -INF
    dw = randn(17, (T, top), std=1.0)
    r = grad.route_experts(logits, top, scoring, renormalize=renormalize, scale=scale)
    assert r.weights.requires_grad and not any(t.requires_grad for t in r[1:])
    assert all(torch.equal(a, b) for a, b in zip(r, mb.route_experts(logits, top, scoring, renormalize=renormalize, scale=scale)))
    g, = torch.autograd.grad(r.weights, logits, dw)
    ref = exact_gradient(logits, r.experts, dw, scoring, renormalize, scale)
    assert g.dtype == dt
    # half a unit of the type; in 32 bits the same half units as a weight's, twice, of the row's largest terms (they cancel)
    span = float((logits.detach().double().masked_fill(torch.isinf(logits), 0.0)).abs().max()) * 4
    size = (dw.double().abs().max(-1, keepdim=True).values * scale * (r.weights.detach().double().max(-1, keepdim=True).values / scale)).clamp_min(1e-30)
    room = torch.finfo(dt).eps / 2 * ref.abs() + (2 * span + 110) * 2.0 ** -24 * 2 * top * size + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    assert ((g.double() - ref).abs() <= room).all()


def test_gradient_against_differences():
    """Central differences of step h of the weights in 32 bits: off by h^2 / 6 times a third derivative (at most 1 for these functions)
    and by the weights' roundings, 100 half units each, over h."""
    logits = randn(18, (4, 12)).requires_grad_()
    dw, v, h = randn(19, (4, 3), std=1.0), randn(20, (4, 12), std=1.0), 2.0 ** -7
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            r = grad.route_experts(logits, 3, scoring, renormalize=renormalize)
            g, = torch.autograd.grad(r.weights, logits, dw)
            up, down = (mb.route_experts(logits.detach() + s * h * v, 3, scoring, renormalize=renormalize) for s in (1, -1))
            same = (up.experts == r.experts).all(-1) & (down.experts == r.experts).all(-1)
            slope = ((up.weights - down.weights).double() * dw.double() / (2 * h)).sum(-1)
            room = dw.double().abs().sum(-1) * (h * h / 6 * v.double().abs().sum(-1) ** 3 + 100 * 2.0 ** -24 / h)
            assert same.any() and ((slope - (g.double() * v.double()).sum(-1)).abs() <= room)[same].all()


def test_gradient_of_rows_without_experts():
    logits = randn(21, (5, 20))
    logits[2] = -INF
    logits[3, 2:] = -INF
    logits.requires_grad_()
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (False, True):
            r = grad.route_experts(logits, 4, scoring, renormalize=renormalize)
            g, = torch.autograd.grad(r.weights, logits, torch.ones_like(r.weights))
            assert torch.isfinite(g).all() and (g[2] == 0).all() and (g[3, 2:] == 0).all()


def test_gradient_modes():
    """No gradient, second order (refused), a backward pass captured into a graph."""
    logits = randn(22, (30, 16)).requires_grad_()
    with torch.no_grad():
        assert not grad.route_experts(logits, 2).weights.requires_grad
    assert not grad.route_experts(logits.detach(), 2).weights.requires_grad
    dw = randn(23, (30, 2))
    g, = torch.autograd.grad(grad.route_experts(logits, 2).weights, logits, dw, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    leaf = logits.detach().clone().requires_grad_()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        torch.autograd.grad(grad.route_experts(leaf, 2).weights, leaf, dw)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            got, = torch.autograd.grad(grad.route_experts(leaf, 2).weights, leaf, dw)
        graph.replay()
    st.synchronize()
    assert torch.equal(got, g.detach())
