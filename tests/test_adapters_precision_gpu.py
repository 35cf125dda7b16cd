"""The inner products of add_adapters are held in the 24 bits of their sums: where the ranks', rows' or adapters' terms cancel, that is what is left."""
import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import ops

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def randn(seed, shape, dtype=torch.float32):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def cancelling(seed, shape, dt, dim):
    """Three tensors along `dim` whose sum is exactly zero: u, -(1 + d) u rounded, and what these two leave, which has fewer digits."""
    u = randn(seed, shape, dt)
    v = (-(1 + 0.3 * randn(seed + 1, shape).abs().clamp_max(2.5)) * u.float()).to(dt)
    w = -(u.double() + v.double())
    assert torch.equal(w.to(dt).double(), w)
    return torch.stack((u, v, w.to(dt)), dim)


def near(got, mass, first, second):
    """What should be zero.  fp32 sums truncated at each term: 2^-23 of the magnitudes' sum each, for the `first` products of an inner product and up to 5 products
    (parts of both operands) for each of the `second` ones of the sum after it; 2^-23 for what is left out there, and 2^-23 for the factor c."""
    t = torch.finfo(got.dtype)
    room = (first + 5 * second + 2) * 2.0 ** -23 * mass
    bad = got.double().abs() - room * (1 + t.eps / 2) - t.smallest_normal * t.eps
    assert (bad <= 0).all(), float((bad / mass.clamp_min(1e-30)).max())


def uneven(seed, shape, dt):
    """Pairs of which the second is far smaller: sums that need all of their digits."""
    return torch.stack((randn(seed, shape, dt), (randn(seed + 1, shape) * 2.0 ** -6).to(dt)), -1)


@pytest.mark.parametrize("dtype", tuple(DTYPES))
@pytest.mark.parametrize("T", (5, 64, 300))
def test_ranks_that_cancel(dtype, T):
    """a's rows add up to zero and b's columns are equal: nothing is left of the sum.  The gradient of x: b's columns add up to zero."""
    dt, N = DTYPES[dtype], 40
    ids = torch.zeros(T, dtype=torch.int64, device="cuda")
    groups = mb.group_rows(ids, 1)
    x, y = uneven(1, (T,), dt), torch.zeros((T, N), dtype=dt, device="cuda")
    a, b = cancelling(3, (1, 2), dt, 1), randn(5, (1, N, 1), dt).expand(1, N, 3).contiguous()
    mass = (x.double().abs() @ a[0].double().abs().sum(0))[:, None] * b[0, :, 0].double().abs()
    near(mb.add_adapters(y, x, a, b, groups), mass, 2, 3)

    a, b, dy = randn(6, (1, 1, N), dt).expand(1, 3, N).contiguous(), cancelling(7, (1, 2), dt, 2), uneven(9, (T,), dt)
    x, s = randn(11, (T, N), dt), torch.tensor([1.3], device="cuda")
    dx, _, _ = mb.add_adapters_grad(dy, x, a, b, groups, ops._add_adapters(dy, x, a, b, groups, s)[1], s)
    mass = 1.3 * (dy.double().abs() @ b[0].double().abs().sum(1))[:, None] * a[0, 0].double().abs()
    near(dx, mass, 2, 3)


@pytest.mark.parametrize("dtype", tuple(DTYPES))
@pytest.mark.parametrize("r", (16, 40, 70))
def test_rows_that_cancel(dtype, r):
    """Three rows of x add up to zero and their dy are the same, and the other way round: gradients of b and a."""
    dt, N, K, L = DTYPES[dtype], 2, 24, 2
    ids = torch.tensor([1, 0, 1, -1, 1], device="cuda")
    rows = [0, 2, 4]
    groups, s = mb.group_rows(ids, L), torch.tensor([0.7, 1.3], device="cuda")
    x, dy = randn(1, (5, K), dt), randn(2, (5, N), dt)
    a, b = randn(3, (L, r, K), dt), randn(4, (L, N, r), dt)
    a[:, :, 1] *= 2.0 ** -6
    b[:, 1] *= 2.0 ** -6
    x[:, 2:] = 0
    x[rows, :2], dy[rows] = cancelling(5, (2,), dt, 0), dy[0].clone()
    _, _, db = mb.add_adapters_grad(dy, x, a, b, groups, ops._add_adapters(dy, x, a, b, groups, s)[1], s)
    mass = 1.3 * dy[0].double().abs()[:, None] * (x[rows].double().abs().sum(0) @ a[1].double().abs().T)
    near(db[1], mass, 2, 3)
    x = randn(7, (5, K), dt)
    x[rows], dy[rows] = x[0].clone(), cancelling(8, (N,), dt, 0)
    _, da, _ = mb.add_adapters_grad(dy, x, a, b, groups, ops._add_adapters(dy, x, a, b, groups, s)[1], s)
    mass = 1.3 * (dy[rows].double().abs().sum(0) @ b[1].double().abs())[:, None] * x[0].double().abs()
    near(da[1], mass, N, 3)


@pytest.mark.parametrize("dtype", tuple(DTYPES))
@pytest.mark.parametrize("r", (4, 33, 70))
def test_infinite_inner_products(dtype, r):
    """An infinity in x (dy) whose products with a (b) have one sign: the sums are the infinities of the formula, for weights of any digits."""
    dt, N, K = DTYPES[dtype], 48, 40
    ids = torch.tensor([0] * 20 + [-1] * 3, device="cuda")
    groups = mb.group_rows(ids, 1)
    y, x, dy = randn(1, (23, N), dt), randn(2, (23, K), dt), randn(3, (23, N), dt)
    a, b = randn(4, (1, r, K), dt).abs() + 0.5, randn(5, (1, N, 1), dt).expand(1, N, r).contiguous()
    b[0, :8] = torch.tensor([1.0, -1.0, 0.5, -3.0, 1.0, 2.0, -256.0, 4.0], dtype=dt, device="cuda")[:, None]
    x[5, 3], x[7, 1] = float("inf"), -float("inf")
    out = mb.add_adapters(y, x, a, b, groups)
    h = x[:20].double() @ a[0].double().T
    ref = y.double()
    ref[:20] += h @ b[0].double().T
    assert torch.isinf(ref[5]).all() and torch.isinf(ref[7]).all()
    for t in (5, 7):
        assert torch.equal(out[t].double(), ref[t])
    others = [0, 4, 6, 8, 22]   # (in float16 some of their results are beyond the type: 70 times 256 times 18)
    assert torch.equal(torch.isfinite(out[others]), torch.isfinite(ref.to(dt)[others]))
    # dy h^T with a row of infinite h: infinities of dy's signs; dy infinite: g a
    x[7, 1] = 0.0
    got = mb.add_adapters_grad(dy, x, a, b, groups, ops._add_adapters(y, x, a, b, groups)[1], None, False, False, True)[2][0]
    assert torch.equal(got.double(), (dy[5].double()[:, None] * float("inf")).expand(N, r))
    dy[9, 0] = float("inf")
    b = b.abs()
    dx = mb.add_adapters_grad(dy, x, a, b, groups, ops._add_adapters(y, x, a, b, groups)[1], None, True, False, False)[0]
    others = [0, 8, 10, 21]
    ref = torch.where(ids[others, None] < 0, 0.0, dy[others].double() @ b[0].double() @ a[0].double())
    assert (dx[9] == float("inf")).all() and torch.equal(torch.isfinite(dx[others]), torch.isfinite(ref.to(dt)))
