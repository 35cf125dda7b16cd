"""grad.grouped_mm in forward mode (refused), under hooks on saved tensors, in checkpoints, and called from several threads' backward passes."""
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.utils.checkpoint import checkpoint

import mlx_b200 as mb
from mlx_b200 import grad, ops
from test_grouped_gpu import randn

pytestmark = pytest.mark.gpu
SIZES = [7, 0, 30, 1]


def problem():
    x, w = randn(1, (38, 72), torch.bfloat16), randn(2, (4, 40, 72), torch.bfloat16)
    dy, n = randn(3, (38, 40), torch.bfloat16), torch.tensor(SIZES, device="cuda")
    return x, w, dy, n, mb.grouped_mm(dy, w, n, False), mb.grouped_mm_dw(dy, x, n)


@pytest.mark.parametrize("requires_grad", (False, True))
@pytest.mark.parametrize("of", ("x", "w"))
def test_forward_mode_is_refused(of, requires_grad):
    """A tangent is never dropped silently."""
    x, w, _, n, _, _ = problem()
    x.requires_grad_(requires_grad)
    with fwd.dual_level():
        t = x if of == "x" else w
        d = fwd.make_dual(t, torch.ones_like(t))
        with pytest.raises(RuntimeError):
            grad.grouped_mm(d if of == "x" else x, d if of == "w" else w, n)


def transposed(t):
    """The same values, laid out otherwise."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else t.clone()


@pytest.mark.parametrize("pack,unpack", ((lambda t: t.cpu(), lambda t: t.cuda()), (transposed, lambda t: t), (lambda t: t, transposed)))
def test_hooks_on_saved_tensors(pack, unpack):
    x, w, dy, n, dx, dw = problem()
    x.requires_grad_(), w.requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        y = grad.grouped_mm(x, w, n)
    got = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(got[0], dx) and torch.equal(got[1], dw)


def test_checkpoint():
    x, w, dy, n, dx, dw = problem()
    x.requires_grad_(), w.requires_grad_()
    checkpoint(lambda x, w: grad.grouped_mm(x, w, n), x, w, use_reentrant=False).backward(dy)
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)


def test_saved_tensors_that_were_overwritten_are_noticed():
    x, w, dy, n, _, _ = problem()
    w.requires_grad_()
    y = grad.grouped_mm(x, w, n)
    x.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward(dy)


def test_backward_passes_of_several_threads():
    x, w, dy, n, dx, dw = problem()
    bad = []

    def work():
        for _ in range(50):
            a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
            grad.grouped_mm(a, b, n).backward(dy)
            if not (torch.equal(a.grad, dx) and torch.equal(b.grad, dw)):
                bad.append(1)

    ts = [threading.Thread(target=work) for _ in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad
    ops.check_status()
