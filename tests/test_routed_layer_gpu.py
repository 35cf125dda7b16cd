"""Routing, rows, products and adapters together, as a layer uses them; and the calls' gradients in every mode of autograd."""
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.utils.checkpoint import checkpoint

import mlx_b200 as mb
from mlx_b200 import grad, ops

pytestmark = pytest.mark.gpu


def randn(seed, shape, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def layer(x, router, up, down, a, b, groups, top, g=grad):
    """A shared projection with the requests' adapters, then experts: what a decoder's block does with them."""
    x = g.add_adapters(x, x, a, b, groups)
    r = g.route_experts(x @ router.T, top, "sigmoid", renormalize=True)
    h = torch.nn.functional.silu(g.grouped_mm(g.dispatch_rows(x, r), up, r.sizes))
    return g.combine_rows(g.grouped_mm(h, down, r.sizes), r), r.experts


def exact(x, router, up, down, a, b, ids, experts):
    c = (ids >= 0).double()[:, None]
    x = x + c * torch.einsum("tnr,tr->tn", b[ids.clamp_min(0)], torch.einsum("trk,tk->tr", a[ids.clamp_min(0)], x))
    s = torch.sigmoid(x @ router.T).gather(1, experts.long())
    e = experts.long()
    h = torch.nn.functional.silu(torch.einsum("tk,tjhk->tjh", x, up[e]))
    return torch.einsum("tj,tjk->tk", s / s.sum(-1, keepdim=True), torch.einsum("tjh,tjkh->tjk", h, down[e]))


@pytest.mark.parametrize("T,dtype", ((1, torch.bfloat16), (37, torch.float16), (300, torch.bfloat16)))
def test_a_layer_and_its_gradients(T, dtype):
    """Against 64 bits with the experts that were chosen.  Every activation is rounded to 16 bits on the way, seven of them in a row:
    off by some units of the whole, where a wrong row, expert or weight makes it about 1."""
    D, H, E, top, L, r = 128, 192, 16, 3, 3, 8
    x, router, up, down = randn(1, (T, D), dtype), randn(2, (E, D), dtype, D ** -0.5), randn(3, (E, H, D), dtype, D ** -0.5), randn(4, (E, D, H), dtype, H ** -0.5)
    a, b = randn(5, (L, r, D), dtype, D ** -0.5), randn(6, (L, D, r), dtype, r ** -0.5)
    ids = torch.randint(-1, L, (T,), generator=torch.Generator().manual_seed(7)).cuda()
    groups = mb.group_rows(ids, L)
    leaves = [t.requires_grad_() for t in (x, router, up, down, a, b)]
    y, experts = layer(*leaves, groups, top)
    dy = randn(8, (T, D), dtype)
    got = torch.autograd.grad(y, leaves, dy)
    exacts = [t.detach().double().requires_grad_() for t in leaves]
    ref = exact(*exacts, ids, experts)
    for p, q in zip((y, *got), (ref, *torch.autograd.grad(ref, exacts, dy.double()))):
        assert (p.double() - q).norm() <= 16 * torch.finfo(dtype).eps * q.norm()
    with torch.no_grad():
        z, again = layer(*leaves, groups, top, mb)
    assert torch.equal(z, y) and torch.equal(again, experts)
    # captured, with other activations and requests under the graph
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st), torch.no_grad():
        static, who = x.detach().clone(), ids.clone()
        layer(static, *leaves[1:], mb.group_rows(who, L), top, mb)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            z, _ = layer(static, *leaves[1:], mb.group_rows(who, L), top, mb)
        static.copy_(x.flip(0)), who.copy_(ids.flip(0))
        graph.replay()
        st.synchronize()
        want, _ = layer(static, *leaves[1:], mb.group_rows(who, L), top, mb)
        st.synchronize()
    assert torch.equal(z, want)
    ops.check_status()


def calls():
    """(what, its leaves, the call) of every operator with a gradient."""
    logits = randn(10, (30, 12), torch.float32)
    r = mb.route_experts(logits, 3)
    ids = torch.tensor([0, 1, -1, 1, 0] * 6, device="cuda")
    groups = mb.group_rows(ids, 2)
    s = torch.tensor([0.5, 2.0], device="cuda")
    x, ys, w = randn(11, (30, 40)), randn(12, (90, 40)), randn(13, (30, 3), torch.float32)
    y, a, b = randn(14, (30, 24)), randn(15, (2, 4, 40)), randn(16, (2, 24, 4))
    return (("route", [logits], lambda l: grad.route_experts(l, 3, renormalize=True).weights),
            ("dispatch", [x], lambda x: grad.dispatch_rows(x, r)),
            ("combine", [ys, w], lambda y, w: grad.combine_rows(y, r._replace(weights=w))),
            ("adapters", [y, x, a, b], lambda y, x, a, b: grad.add_adapters(y, x, a, b, groups, s)))


def gradients(leaves, call):
    leaves = [t.clone().requires_grad_() for t in leaves]
    y = call(*leaves)
    return torch.autograd.grad(y, leaves, randn(17, y.shape, y.dtype)), y


def same(p, q):
    assert len(p) == len(q) and all(torch.equal(a, b) for a, b in zip(p, q))


@pytest.mark.parametrize("i", range(4))
def test_forward_mode_is_refused(i):
    _, leaves, call = calls()[i]
    for k in range(len(leaves)):
        with fwd.dual_level():
            args = list(leaves)
            args[k] = fwd.make_dual(args[k], torch.ones_like(args[k]))
            with pytest.raises(RuntimeError):
                call(*args)


def turned(t):
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t.clone()


@pytest.mark.parametrize("i", range(4))
@pytest.mark.parametrize("pack,unpack", ((lambda t: t.cpu(), lambda t: t.cuda()), (turned, lambda t: t), (lambda t: t, turned)))
def test_hooks_on_saved_tensors(i, pack, unpack):
    _, leaves, call = calls()[i]
    ref, y = gradients(leaves, call)
    leaves = [t.clone().requires_grad_() for t in leaves]
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        z = call(*leaves)
    same(torch.autograd.grad(z, leaves, randn(17, y.shape, y.dtype)), ref)


@pytest.mark.parametrize("i", range(4))
def test_checkpoints_views_broadcasts_and_second_order(i):
    _, leaves, call = calls()[i]
    ref, y = gradients(leaves, call)
    dy = randn(17, y.shape, y.dtype)
    leaves = [t.clone().requires_grad_() for t in leaves]
    same(torch.autograd.grad(checkpoint(call, *leaves, use_reentrant=False), leaves, dy), ref)
    same(torch.autograd.grad(call(*leaves), leaves, turned(dy)), ref)
    others = [turned(t.detach()).requires_grad_() for t in leaves]   # the Python form, where strides differ
    same(torch.autograd.grad(call(*others), others, dy), ref)
    same(torch.autograd.grad(call(*leaves).sum(), leaves), torch.autograd.grad(call(*leaves), leaves, torch.ones_like(dy)))
    first = torch.autograd.grad(call(*leaves), leaves, dy, create_graph=True)
    same([t.detach() for t in first], ref)
    with pytest.raises(RuntimeError):
        sum(t.float().sum() for t in first if t is not dy).backward()


@pytest.mark.parametrize("i", range(4))
def test_saved_tensors_that_were_overwritten_are_noticed(i):
    what, leaves, call = calls()[i]
    if what == "dispatch":
        pytest.skip("its gradient does not read x")
    leaves = [t.clone().requires_grad_() for t in leaves]
    y = call(*leaves)
    with torch.no_grad():
        leaves[1 if what == "adapters" else 0].mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, leaves, torch.ones_like(y))


def test_backward_passes_of_several_threads():
    all_calls = calls()
    refs = [gradients(leaves, call)[0] for _, leaves, call in all_calls]
    bad = []

    def work():
        for _ in range(20):
            for (_, leaves, call), ref in zip(all_calls, refs):
                if not all(torch.equal(p, q) for p, q in zip(gradients(leaves, call)[0], ref)):
                    bad.append(1)

    ts = [threading.Thread(target=work) for _ in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_gradients_that_are_not_asked_for_are_not_computed():
    """Launches of a backward pass: as many kernels as what is wanted needs."""
    from mlx_b200 import _lib
    _, leaves, call = calls()[3]
    _, h = ops._add_adapters(*leaves, mb.group_rows(torch.tensor([0, 1, -1, 1, 0] * 6, device="cuda"), 2))
    count = lambda *wanted: (lambda n: (mb.add_adapters_grad(randn(17, (30, 24)), *leaves[1:], mb.group_rows(torch.tensor([0, 1, -1, 1, 0] * 6, device="cuda"), 2), h, None,
                                                             *wanted), _lib.load().b200q_launch_count() - n)[1])(_lib.load().b200q_launch_count())
    one = count(False, False, True)
    assert count(True, True, True) == one + 3 and count(True, False, False) == one + 1 and count(False, True, False) == one + 1
