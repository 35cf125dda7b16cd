"""A sum so long that the wait for its tile outlasts the usual limit of a wait."""
import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import ops

pytestmark = pytest.mark.gpu


def test_a_tile_of_thirty_million_stages():
    """Two vectors of 1.9e9 elements (3.8 GB each): one tile, too many steps to be cut, some seconds of one pair of blocks.  All but a
    thousand products are zero and their sum is exact."""
    K = 1_900_000_000
    x, w = (torch.zeros(K, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    at = torch.arange(1000, device="cuda") * 1_899_998 + 1234
    at[-1] = K - 1
    x[at], w[at] = (torch.arange(1000, device="cuda") % 16).bfloat16(), 2.0
    y = mb.grouped_mm(x.view(1, K), w.view(1, 1, K), torch.tensor([1], device="cuda"))
    ops.check_status()
    assert y.item() == torch.tensor(float(2 * (torch.arange(1000) % 16).sum())).bfloat16().item()
