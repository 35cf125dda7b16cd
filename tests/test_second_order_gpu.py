"""Gradients of the gradients of quantized_matmul."""
import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import grad
from test_grad_gpu import dense_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ("native", "python"))
@pytest.mark.parametrize("transpose", (True, False))
def test_qmm_with_frozen_weights(transpose, form):
    """dx = dy W is linear in dy: what comes back through it is the product itself."""
    torch.manual_seed(1)
    M, N, K = 24, 256, 384
    q = mb.quantize(torch.randn((N, K) if transpose else (K, N), device="cuda").bfloat16())
    x = torch.randn(M, K, device="cuda").bfloat16()
    if form == "python":
        x = x.t().contiguous().t()
    mb.quantized_matmul(torch.zeros(512, N, device="cuda", dtype=torch.bfloat16), *q, transpose=not transpose)   # (scratch is there)
    mb.quantized_matmul(torch.zeros(512, K, device="cuda", dtype=torch.bfloat16), *q, transpose=transpose)
    x.requires_grad_()
    dy = torch.randn(M, N, device="cuda").bfloat16().requires_grad_()
    (gx,) = torch.autograd.grad(grad.quantized_matmul(x, *q, transpose), x, dy, create_graph=True)
    assert torch.equal(gx, mb.quantized_matmul(dy.detach(), *q, transpose=not transpose))
    a, c = torch.randn_like(gx).detach(), torch.randn_like(dy).detach()
    ((gx * a).sum() + (dy * c).sum()).backward()
    assert torch.equal(dy.grad, mb.quantized_matmul(a.contiguous(), *q, transpose=transpose) + c)


@pytest.mark.parametrize("transpose", (True, False))
def test_qmm_with_scales_and_biases(transpose):
    torch.manual_seed(2)
    M, N, K, g, bits = 8, 256, 128, 64, 4
    wq, s, b = mb.quantize(torch.randn((N, K) if transpose else (K, N), device="cuda"), g, bits)
    x, c = torch.randn(M, K, device="cuda"), torch.randn(M, N, device="cuda")
    u = [torch.randn_like(t) for t in (x, s, b)]
    codes = mb.dequantize(wq, torch.ones_like(s), torch.zeros_like(b), g, bits).double()

    def second(f, *args):
        args = [t.requires_grad_() for t in args]
        first = torch.autograd.grad(f(*args[:3]), args[:3], args[3], create_graph=True)
        return torch.autograd.grad(sum((p * q.to(p.dtype)).sum() for p, q in zip(first, u)), args)

    got = second(lambda x, s, b: grad.quantized_matmul(x, wq, s, b, transpose, g, bits), *(t.clone() for t in (x, s, b, c)))
    ref = second(lambda x, s, b: dense_reference(x, codes, s, b, transpose, g), *(t.double() for t in (x, s, b, c)))
    for p, r in zip(got, ref):   # fp32 sums, TF32 allowed in the dense products (as for the first order)
        assert p.shape == r.shape and float((p.double() - r).abs().max()) <= 2e-3 * float(r.abs().max())
