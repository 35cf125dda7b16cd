"""Gradients of grad.grouped_mm's gradients: exact, against the same products, through the native and the Python form."""
import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import grad, ops
from test_grouped_gpu import randn

pytestmark = pytest.mark.gpu
SIZES, N, K = [7, 0, 30, 1], 40, 72


def problem(form, transpose):
    """x, w, dy that require gradients.  The native form takes contiguous operands; a transposed view goes through the Python form."""
    T, bf = sum(SIZES), torch.bfloat16
    x, w = randn(1, (T, K), bf), randn(2, (len(SIZES), N, K) if transpose else (len(SIZES), K, N), bf)
    if form == "python":
        x = x.t().contiguous().t()
    dy, n = randn(3, (T, N), bf), torch.tensor(SIZES, device="cuda")
    mb.grouped_mm_dw(dy, x, n, transpose)   # (the largest scratch is there: the native form takes ordinary calls)
    return [t.requires_grad_() for t in (x, w, dy)] + [n]


@pytest.mark.parametrize("transpose", (True, False))
@pytest.mark.parametrize("form", ("native", "python"))
def test_gradients_of_gradients(form, transpose):
    """dx = dy w and dw = dy^T x are products of two factors each; what comes back through them is the same products."""
    x, w, dy, n = problem(form, transpose)
    gx, gw = torch.autograd.grad(grad.grouped_mm(x, w, n, transpose), (x, w), dy, create_graph=True)
    X, W, D = x.detach(), w.detach(), dy.detach()
    assert torch.equal(gx, mb.grouped_mm(D, W, n, not transpose)) and torch.equal(gw, mb.grouped_mm_dw(D, X, n, transpose))
    a, b = randn(4, gx.shape, gx.dtype), randn(5, gw.shape, gw.dtype)
    ((gx * a).sum() + (gw * b).sum()).backward()
    assert torch.equal(w.grad, mb.grouped_mm_dw(D, a, n, transpose))
    assert torch.equal(x.grad, mb.grouped_mm(D, b, n, not transpose))
    assert torch.equal(dy.grad, mb.grouped_mm(a, W, n, transpose) + mb.grouped_mm(X, b, n, transpose))
    ops.check_status()


@pytest.mark.parametrize("form", ("native", "python"))
def test_a_gradient_penalty_reaches_the_weights(form):
    """The cotangent needs no gradient here, and y itself is part of the loss: nothing but the weights' gradient tells."""
    x, w, _, n = problem(form, True)
    y = grad.grouped_mm(x, w, n)
    one = torch.ones_like(y)
    (gx,) = torch.autograd.grad(y, x, one, create_graph=True)
    a = randn(4, gx.shape, gx.dtype)
    (y.sum() + (gx * a).sum()).backward()
    assert torch.equal(w.grad, mb.grouped_mm_dw(one, x.detach(), n) + mb.grouped_mm_dw(one, a, n))
    assert torch.equal(x.grad, gx)


def test_third_order():
    x, w, dy, n = problem("native", True)
    gx, gw = torch.autograd.grad(grad.grouped_mm(x, w, n), (x, w), dy, create_graph=True)
    a, b = randn(4, gx.shape, gx.dtype).requires_grad_(), randn(5, gw.shape, gw.dtype)
    (dw,) = torch.autograd.grad((gx * a).sum(), w, create_graph=True)   # dy^T a
    (da,) = torch.autograd.grad((dw * b).sum(), a)
    assert torch.equal(da, mb.grouped_mm(dy.detach(), b, n, False))
