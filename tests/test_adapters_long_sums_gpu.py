"""Sums over many rows and wide inputs are not truncated term by term: all terms are positive, and what every truncation takes away would add up."""
import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import ops

pytestmark = pytest.mark.gpu


def positive(seed, shape, size=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return ((torch.rand(shape, generator=g, device="cuda") * 0.5 + 0.5) * size).half()


def mean_error(got, ref, rounded):
    """The results' mean relative error.  Of n results each is rounded to float16, off by 2^-12 at random, which leaves six times 2^-12 / sqrt(3 n) at most; and sums of `rounded` nearest roundings in
    fp32, 2^-24 each, six times 2^-24 sqrt(rounded) if they were all the same."""
    e = float(((got.double() - ref) / ref).mean())
    assert abs(e) <= 6 * (2.0 ** -12 / (3 * ref.numel()) ** 0.5 + 2.0 ** -24 * rounded ** 0.5), e


@pytest.mark.parametrize("r", (8, 64))
def test_gradients_of_an_adapter_of_many_rows(r):
    T, L, N, K = 200000, 300, 128, 64
    ids = torch.zeros(T, dtype=torch.int64, device="cuda")
    x, dy, a, b = positive(1, (T, K)), positive(2, (T, N), 2.0 ** -8), positive(3, (L, r, K), 2.0 ** -6), positive(4, (L, N, r), 2.0 ** -4)
    groups = mb.group_rows(ids, L)
    _, da, db = mb.add_adapters_grad(dy, x, a, b, groups, None, None, False)
    h, g = x.double() @ a[0].double().T, dy.double() @ b[0].double()
    mean_error(db[0], dy.double().T @ h, T / 16 * 3)
    mean_error(da[0], g.T @ x.double(), T / 16 * 3)


@pytest.mark.parametrize("tall", (False, True))
def test_long_inner_products(tall):
    T, C, n, r = 8, 1 << 22, 2048, 1
    ids = torch.zeros(T, dtype=torch.int64, device="cuda")
    groups, c = mb.group_rows(ids, 1), torch.tensor([2.0 ** -21], device="cuda")
    x, w, v = positive(1, (T, C)), positive(2, (1, C), 1.0), positive(3, (1, n))
    ref = 2.0 ** -21 * (x.double() @ w[0].double())[:, None] * v[0].double()
    if tall:   # the gradient of x: sums along b's columns
        got = mb.add_adapters_grad(x, torch.zeros((T, n), device="cuda").half(), v.reshape(1, 1, n), w.reshape(1, C, 1), groups, None, c, True, False, False)[0]
    else:
        got = mb.add_adapters(torch.zeros((T, n), device="cuda").half(), x, w.reshape(1, 1, C), v.reshape(1, n, 1), groups, c)
    mean_error(got, ref, C / 32)


def test_many_ranks():
    T, K, N, r = 64, 64, 512, 4096
    ids = torch.zeros(T, dtype=torch.int64, device="cuda")
    groups, c = mb.group_rows(ids, 1), torch.tensor([2.0 ** -8], device="cuda")
    x, a, b = positive(1, (T, K)), positive(2, (1, r, K), 2.0 ** -6), positive(3, (1, N, r))
    got = mb.add_adapters(torch.zeros((T, N), device="cuda").half(), x, a, b, groups, c)
    mean_error(got, 2.0 ** -8 * (x.double() @ a[0].double().T) @ b[0].double().T, r / 16)
