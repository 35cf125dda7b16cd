"""Gradients of the adapters that do without the forward pass's inner products, and what they are where the caller has none."""
import os
import shutil
import subprocess

import pytest
import torch

import mlx_b200 as mb
from mlx_b200 import _lib, ops


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_the_cpp_shim(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe, libdir = str(tmp_path / "check"), os.path.dirname(_lib.LIB_PATH)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(root, "include"), os.path.join(root, "tests", "adapters_shim_check.cpp"), "-o", exe,
                    "-L", libdir, "-lb200q", f"-Wl,-rpath,{libdir}"], check=True, capture_output=True, text=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and "SHIM-OK" in res.stdout, res.stdout + res.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_gradients_without_inner_products(dtype):
    g = torch.Generator("cuda").manual_seed(1)
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(dtype)
    ids = torch.tensor([0, 1, -1, 1, 0] * 30, device="cuda")
    groups, s = mb.group_rows(ids, 2), torch.tensor([0.5, 2.0], device="cuda")
    y, x, a, b, dy = rand(150, 72), rand(150, 40), rand(2, 20, 40), rand(2, 72, 20), rand(150, 72)
    ref = mb.add_adapters_grad(dy, x, a, b, groups, ops._add_adapters(y, x, a, b, groups, s)[1], s)
    assert all(torch.equal(p, q) for p, q in zip(mb.add_adapters_grad(dy, x, a, b, groups, scales=s), ref))
    for i, wanted in enumerate(((True, False, False), (False, True, False), (False, False, True))):
        assert torch.equal(mb.add_adapters_grad(dy, x, a, b, groups, None, s, *wanted)[i], ref[i])
    with pytest.raises(ValueError):
        mb.add_adapters_grad(dy, x, a, b, groups, torch.empty((150, 2, 32), dtype=torch.bfloat16, device="cuda"), s)
