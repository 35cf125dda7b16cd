"""A backward pass of grad.grouped_mm computes what it is asked for."""
import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import grad

pytestmark = pytest.mark.gpu


def test_the_gradient_of_one_operand_leaves_the_other_s_out():
    """dw of these experts takes 64 MB, dx 2 KB: the peak of allocated memory tells whether dw was made."""
    bf = dict(dtype=torch.bfloat16, device="cuda")
    x, w = torch.ones(8, 128, **bf).requires_grad_(), torch.ones(4, 65536, 128, **bf).requires_grad_()
    n = torch.tensor([2, 2, 2, 2], device="cuda")
    dy = torch.ones(8, 65536, **bf)
    mb.grouped_mm_dw(dy, x, n), mb.grouped_mm(dy, w, n, False)   # (scratch is there)
    y = grad.grouped_mm(x, w, n)

    def peak(of):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = torch.autograd.grad(y, of, dy, retain_graph=True)
        return torch.cuda.max_memory_allocated() - before, got

    used, (dx,) = peak([x])
    assert used < 1 << 20, used
    used, (dw,) = peak([w])
    assert used >= dw.numel() * 2
    used, both = peak([x, w])
    assert torch.equal(both[0], dx) and torch.equal(both[1], dw)
