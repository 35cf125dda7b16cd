"""Both sides of the rules that choose between forms of the routing and row kernels: one block or several, a block or a warp for a pair, four or eight blocks of a
cluster, tiles shared evenly or not."""
import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import ops
from test_adapters_gpu import exact, near as near_adapters, problem
from test_routing_gpu import check, randn as logits_of
from test_rows_gpu import near, plain, randn, routed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", (16, 17, 24, 25, 33, 47, 48, 49))
@pytest.mark.parametrize("E,top,groups", ((1, 1, 1), (8, 2, 1), (32, 4, 4), (33, 5, 3), (128, 8, 1), (129, 8, 1), (256, 8, 8)))
def test_one_block_and_several(T, E, top, groups):
    logits = logits_of(T, (T, E))
    logits[3] = -float("inf")
    logits[T // 2, E // 2:] = -float("inf")
    for bias in (None, logits_of(2, (E,), std=0.2)):
        check(logits, top, bias, scoring="sigmoid", groups=groups, top_groups=max(1, groups // 2), renormalize=True)


@pytest.mark.parametrize("T,top,D,dtype", ((70, 6, 255, torch.bfloat16), (60, 6, 255, torch.bfloat16), (520, 6, 2047, torch.float16), (500, 6, 2047, torch.float16), (300, 4, 8191, torch.bfloat16),
                                           (9, 2, 7, torch.float32), (800, 4, 1021, torch.float32)))
def test_gradients_of_rows_off_16_bytes(T, top, D, dtype):
    r = routed(1, T, 16, top, 0.3)
    y, dy, w = randn(2, (T * top, D), dtype), randn(3, (T, D), dtype), randn(4, (T, top))
    r = r._replace(weights=w)
    used = int(r.sizes.sum())
    y[used:] = float("nan")
    has, yp = plain(r, None, y, w)
    dys, dw = mb.combine_rows_grad(dy, y, r)
    token, pair = r.order[:used].long() // top, r.order[:used].long()
    near(dys[:used], w.double().flatten()[pair][:, None] * dy.double()[token], torch.zeros((), device="cuda"), 0)
    assert (dys[used:] == 0).all() and (dw[~has] == 0).all()
    near(dw, torch.einsum("td,tjd->tj", dy.double(), yp), torch.einsum("td,tjd->tj", dy.double().abs(), yp.abs()), D)


@pytest.mark.parametrize("T,L,r,N,K", ((2048, 4, 16, 512, 4096), (1024, 1, 64, 512, 4096), (512, 1, 64, 4096, 512), (30, 40, 16, 300, 2048)))
def test_blocks_of_a_cluster(T, L, r, N, K):
    ids = torch.randint(-1, L, (T,), generator=torch.Generator().manual_seed(5)).cuda()
    y, x, a, b, s = problem(6, ids, L, r, N, K, torch.bfloat16)
    groups = mb.group_rows(ids, L)
    out, h = ops._add_adapters(y, x, a, b, groups, s)
    near_adapters(out, *exact(ids, y, x, a, b, s), K + r)
    dx, _, _ = mb.add_adapters_grad(y, x, a, b, groups, h, s, True, False, False)
    near_adapters(dx, *exact(ids, y, x, a, b, s, y)[0], N + r)


@pytest.mark.parametrize("N,dtype", ((14336, torch.bfloat16), (14300, torch.float16), (4096, torch.bfloat16)))
@pytest.mark.parametrize("last", (0.0, 0.9))
@pytest.mark.parametrize("r", (20, 64))
def test_tiles_shared_evenly_and_not(N, dtype, last, r):
    T, L, K = 8192 if N > 5000 else 16000, 6, 64
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(-1, L, (T,), generator=g)
    ids[torch.rand(T, generator=g) < last] = -1
    ids = ids.cuda()
    y, x, a, b, s = problem(8, ids, L, r, N, K, dtype)
    groups = mb.group_rows(ids, L)
    out = mb.add_adapters(y, x, a, b, groups, s)
    near_adapters(out, *exact(ids, y, x, a, b, s), K + r)
    place = y.clone()
    mb.add_adapters(place, x, a, b, groups, s, out=place)
    assert torch.equal(place, out)
