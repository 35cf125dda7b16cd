"""Ranks of groups whose keys are far larger than their sums, or whose sums pass float32's range: the order of 64 bits."""
import numpy as np
import pytest
import torch

import mlx_b200 as mb
import routing_plain as plain

pytestmark = pytest.mark.gpu


def check(logits, top, bias, **kw):
    r = mb.route_experts(logits, top, bias=bias, **kw)
    f64 = lambda t: t.double().cpu().numpy()
    ref = plain.route(f64(logits), top, bias=f64(bias), **kw)
    for got, want, name in zip(r[1:], ref[1:], r._fields[1:]):
        assert np.array_equal(got.cpu().numpy(), want), name


@pytest.mark.parametrize("T", (9, 700))
@pytest.mark.parametrize("size", (30.0, 100.0, 1000.0, 1e5))
@pytest.mark.parametrize("scoring", ("sigmoid", "softmax"))
def test_keys_of_opposite_signs(T, size, scoring):
    """Every group has a key of about +size and one of about -size, whose roundings are larger than the distances of the groups' sums."""
    G = 8
    g = torch.Generator().manual_seed(int(size))
    if scoring == "sigmoid":
        a = torch.randn((T, G), generator=g, dtype=torch.float64)
        s = (1.0 - torch.sigmoid(a) + size * 2.0 ** -24 * torch.randn((T, G), generator=g, dtype=torch.float64)).clamp(0.01, 0.99)
        logits = torch.stack((a, torch.logit(s)), -1)
    else:   # shares of the groups, then of their two experts
        share = (1.0 / G + size * 2.0 ** -24 * torch.randn((T, G), generator=g, dtype=torch.float64)).clamp(0.01, 0.9)
        part = torch.rand((T, G), generator=g, dtype=torch.float64) * 0.8 + 0.1
        logits = torch.stack((share * part, share * (1 - part)), -1).log()
    bias = torch.tensor([size, -size]).repeat(G)
    check(logits.reshape(T, 2 * G).float().cuda(), 5, bias.cuda(), scoring=scoring, groups=G, top_groups=3, group_best=2)
    check(logits.reshape(T, 2 * G).float().cuda(), 5, bias.cuda(), scoring=scoring, groups=G, top_groups=3, group_best=1)


@pytest.mark.parametrize("T", (5, 300))
def test_one_large_group_among_small_ones(T):
    """A group that is neither the last one kept nor the next by its rounded sum, but could be either by its true one."""
    G, n = 6, 4
    g = torch.Generator().manual_seed(3)
    logits = torch.randn((T, G * n), generator=g)
    bias = 0.1 * torch.randn(G * n, generator=g)
    bias[n], bias[n + 1:2 * n] = 3e6, -3e6
    for best in (1, 2):
        check(logits.cuda(), 5, bias.cuda(), scoring="sigmoid", groups=G, top_groups=3, group_best=best)


@pytest.mark.parametrize("T", (1, 40))
@pytest.mark.parametrize("sign", (-1.0, 1.0))
def test_sums_beyond_float32(T, sign):
    """Biases of about the largest and the lowest float32: two of them add up to a number of 64 bits, and to infinities of 32."""
    logits = torch.randn((T, 8), generator=torch.Generator().manual_seed(4)).cuda()
    least = torch.finfo(torch.float32).min
    bias = torch.tensor([least, least, -3.0e38, -3.0e38, 0.0, 0.1, -3.2e38, -3.2e38], device="cuda") * -sign
    for top_groups in (1, 2, 3):
        for scoring in ("sigmoid", "softmax"):
            check(logits, 2 * top_groups, bias, scoring=scoring, groups=4, top_groups=top_groups, group_best=2)


@pytest.mark.parametrize("low", (-1e9, float(torch.finfo(torch.float32).min), -float("inf")))
def test_masked_experts(low):
    """Experts that a bias takes out, whole groups of them and parts."""
    G, n, T = 8, 8, 200
    g = torch.Generator().manual_seed(5)
    logits, bias = torch.randn((T, G * n), generator=g).cuda(), 0.1 * torch.randn(G * n, generator=g)
    bias[:2 * n], bias[3 * n + 1:4 * n], bias[5 * n:5 * n + 3] = low, low, low
    for best in (1, 2):
        for top_groups in (2, 5, 7):
            check(logits, 6, bias.cuda(), scoring="sigmoid", groups=G, top_groups=top_groups, group_best=best)
