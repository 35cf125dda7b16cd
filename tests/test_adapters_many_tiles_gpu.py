"""The second product where its blocks count the tiles that have rows and share them, in the forms that other tests do not bring there: more than 64 ranks, and
the gradient of x."""
import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import ops
from test_adapters_gpu import exact, near, problem, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("last", (0.0, 0.9))
@pytest.mark.parametrize("T,N,K,r", ((16000, 2600, 64, 66), (16000, 2597, 60, 130), (9000, 64, 8200, 4), (9000, 60, 8197, 33), (9000, 64, 8200, 72), (9000, 72, 8203, 72)))
def test_sum_and_gradient_of_x(T, N, K, r, last, dtype):
    """Forward with wide results, gradients of a wide x; rows of 16 bytes and odd ones; few and most rows without an adapter."""
    g = torch.Generator().manual_seed(31)
    ids = torch.randint(-1, 3, (T,), generator=g)
    ids[torch.rand(T, generator=g) < last] = -1
    ids = ids.cuda()
    y, x, a, b, s = problem(32, ids, 4, r, N, K, dtype)
    groups = mb.group_rows(ids, 4)
    out, h = ops._add_adapters(y, x, a, b, groups, s)
    near(out, *exact(ids, y, x, a, b, s), K + r)
    place = y.clone()
    mb.add_adapters(place, x, a, b, groups, s, out=place)
    assert torch.equal(place, out)
    dy = randn(33, (T, N), dtype)
    dx, _, _ = mb.add_adapters_grad(dy, x, a, b, groups, h, s, True, False, False)
    near(dx, *exact(ids, y, x, a, b, s, dy)[0], N + r)
    assert (dx[ids < 0] == 0).all()
