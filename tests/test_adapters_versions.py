"""A sum in place counts as one change of its tensor, and a call that is refused as none: a graph that has kept the tensor stays usable."""
import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import _lib


def operands(dev, T=5, L=2, r=4, N=8, K=16, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(1)
    rand = lambda *shape: torch.randn(shape, generator=g).to(dtype).to(dev)
    return rand(T, N), rand(T, K), rand(L, r, K), rand(L, N, r)


def test_a_call_that_is_refused_changes_nothing():
    y, x, a, b = operands("cpu")
    tables = lambda T: mb.RowGroups(*(torch.zeros(s, dtype=torch.int32) for s in ((2,), (3,), (T,), (_lib.load().b200q_group_rows_tiles(T, 2), 4))))
    w = torch.ones_like(y).requires_grad_()
    z = y * w
    for error, groups, a2 in ((ValueError, tables(4), a), (ValueError, tables(5), a.float()), (ValueError, tables(5), a[:1]), (RuntimeError, tables(5), a)):   # (no CUDA)
        for out in (y, y.clone()):
            before = out._version
            with pytest.raises(error):
                mb.add_adapters(y, x, a2, b, groups, out=out)
            assert out._version == before
    z.sum().backward()
    assert torch.equal(w.grad, y)


@pytest.mark.gpu
def test_versions_on_the_device():
    y, x, a, b = operands("cuda")
    ids = torch.tensor([0, 1, -1, 1, 0], device="cuda")
    groups, s = mb.group_rows(ids, 2), torch.ones(2, device="cuda")
    w = torch.ones_like(y).requires_grad_()
    z = y * w
    before, was = y._version, y.clone()
    with pytest.raises(ValueError):
        mb.add_adapters(y, x, a, b, mb.group_rows(ids[:4], 2), s, out=y)
    with pytest.raises(ValueError):
        mb.add_adapters(y, x.float(), a, b, groups, s, out=y)
    with pytest.raises(RuntimeError):
        mb.add_adapters(y, x, a.new_zeros((2, 4097, 16)), b.new_zeros((2, 8, 4097)), groups, s, out=y)   # too many ranks
    assert y._version == before and torch.equal(y, was)
    z.sum().backward()
    assert torch.equal(w.grad, was)
    mb.add_adapters(y, x, a, b, groups, s, out=y)
    assert y._version == before + 1
    mb.add_adapters(y, x, a, b, groups, s.double(), out=y)
    assert y._version == before + 2
    with torch.inference_mode():
        t, u = was.clone(), was.clone()
    mb.add_adapters(t, x, a, b, groups, s, out=t)
    mb.add_adapters(u, x, a, b, groups, s.double(), out=u)
    assert torch.equal(t, u) and torch.equal(t, mb.add_adapters(was, x, a, b, groups, s))
