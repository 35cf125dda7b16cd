"""A mixture-of-experts layer, trained in bfloat16 and then served with 4-bit weights and activations.

    python examples/moe_layer.py [--tokens 2048] [--experts 8] [--top 2] [--width 1024] [--hidden 2048] [--steps 20] [--mode nvfp4]

Tokens are sorted by expert once; both projections, their gradients and the 4-bit products then work on rows sorted by
expert with the experts' row counts on the device: no padding, no capacity, no synchronisation with the host.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import mlx_b200 as mb  # noqa: E402
from mlx_b200 import grad  # noqa: E402


def route(logits, top):
    """-> (rows of the tokens in expert order, their weights, rows per expert)."""
    weight, expert = torch.softmax(logits.float(), -1).topk(top, -1)
    order = expert.flatten().argsort(stable=True)
    sizes = torch.zeros(logits.shape[-1], dtype=torch.int64, device=logits.device)
    sizes.scatter_add_(0, expert.flatten(), torch.ones_like(expert.flatten()))
    return order // top, weight.flatten()[order], sizes


class Layer:
    def __init__(self, experts, width, hidden, gen):
        def weights(*shape):
            return (torch.randn(shape, generator=gen, device="cuda") / shape[-1] ** 0.5).to(torch.bfloat16).requires_grad_()

        self.router, self.up, self.down = weights(experts, width), weights(experts, hidden, width), weights(experts, width, hidden)

    def __call__(self, x, top):
        rows, weight, sizes = route(x @ self.router.T, top)
        h = torch.nn.functional.silu(grad.grouped_mm(x[rows], self.up, sizes))
        y = grad.grouped_mm(h, self.down, sizes) * weight[:, None].to(x.dtype)
        return torch.zeros_like(x).index_add(0, rows, y)

    def parameters(self):
        return [self.router, self.up, self.down]


class Served:
    """The same layer with its experts in a microscaled 4-bit mode."""

    def __init__(self, layer, mode, x):
        self.mode, self.router = mode, layer.router.detach()
        self.scale = (lambda t: (t.detach().abs().amax().float() / (448 * 6)).reshape(1)) if mode == "nvfp4" else (lambda t: None)
        self.weights = []
        for w in (layer.up, layer.down):
            g = self.scale(w)
            self.weights.append((*mb.quantize(w.detach(), mode=mode, global_scale=g), g))
        # scales of the activations, as calibration on x finds them
        rows, _, sizes = route(x @ self.router.T, 1)
        self.gx = self.scale(x)
        self.gh = self.scale(torch.nn.functional.silu(mb.grouped_mm(x[rows], layer.up.detach(), sizes)))

    def __call__(self, x, top):
        rows, weight, sizes = route(x @ self.router.T, top)
        (uq, us, ug), (dq, ds, dg) = self.weights
        h = torch.nn.functional.silu(mb.grouped_qqmm(x[rows], uq, us, sizes, mode=self.mode, global_scale_x=self.gx, global_scale_w=ug))
        y = mb.grouped_qqmm(h, dq, ds, sizes, mode=self.mode, global_scale_x=self.gh, global_scale_w=dg) * weight[:, None].to(x.dtype)
        return torch.zeros_like(x).index_add(0, rows, y)


def run(tokens=2048, experts=8, top=2, width=1024, hidden=2048, steps=20, mode="nvfp4", seed=0):
    """-> (first loss, last loss, relative error of the served layer on new tokens)."""
    gen = torch.Generator("cuda").manual_seed(seed)
    layer = Layer(experts, width, hidden, gen)
    opt = torch.optim.Adam(layer.parameters(), lr=2e-3)
    target = torch.randn(width, width, generator=gen, device="cuda") / width ** 0.5
    x = torch.randn(tokens, width, generator=gen, device="cuda").to(torch.bfloat16)
    losses = []
    for _ in range(steps):
        opt.zero_grad()
        loss = (layer(x, top).float() - x.float() @ target).square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    served = Served(layer, mode, x)
    x = torch.randn(tokens // 2 + 1, width, generator=gen, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        a, b = layer(x, top).float(), served(x, top).float()
    return losses[0].item(), losses[-1].item(), ((a - b).norm() / a.norm()).item()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("tokens", 2048), ("experts", 8), ("top", 2), ("width", 1024), ("hidden", 2048), ("steps", 20)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--mode", choices=("mxfp4", "nvfp4"), default="nvfp4")
    first, last, error = run(**vars(ap.parse_args()))
    print(f"loss {first:.4f} -> {last:.4f}; 4-bit layer's output off by {error:.3f} of its norm")
