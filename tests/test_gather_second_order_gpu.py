"""Gradients of the gradients of gather_qmm."""
import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import grad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("transpose", (True, False))
def test_gather_qmm(transpose):
    torch.manual_seed(3)
    E, B, M, N, K, g, bits = 4, 6, 2, 256, 128, 64, 4
    wq, s, b = mb.quantize(torch.randn((E, N, K) if transpose else (E, K, N), device="cuda"), g, bits)
    lhs, rhs = (torch.tensor(i, device="cuda") for i in ([0, 0, 3, 5, 5, 5, 2], [1, 3, 0, 1, 1, 1, 3]))
    x, c = torch.randn(B, M, K, device="cuda"), torch.randn(7, M, N, device="cuda")
    u = [torch.randn_like(t) for t in (x, s, b)]
    codes = mb.dequantize(wq, torch.ones_like(s), torch.zeros_like(b), g, bits).double()

    def plain(x, s, b):
        w = (codes.unflatten(-1, (-1, g)) * s.unsqueeze(-1) + b.unsqueeze(-1)).flatten(-2)
        return torch.stack([x[l] @ (w[r].transpose(0, 1) if transpose else w[r]) for l, r in zip(lhs.tolist(), rhs.tolist())])

    def second(f, *args):
        args = [t.requires_grad_() for t in args]
        first = torch.autograd.grad(f(*args[:3]), args[:3], args[3], create_graph=True)
        return torch.autograd.grad(sum((p * q.to(p.dtype)).sum() for p, q in zip(first, u)), args)

    got = second(lambda x, s, b: grad.gather_qmm(x, wq, s, b, lhs, rhs, transpose, g, bits), *(t.clone() for t in (x, s, b, c)))
    ref = second(plain, *(t.double() for t in (x, s, b, c)))
    for p, r in zip(got, ref):
        assert p.shape == r.shape and float((p.double() - r).abs().max()) <= 2e-3 * float(r.abs().max())
