"""The C++ shim's checks of what the microscaled and grouped functions write into, on the host alone."""
import os
import shutil
import subprocess

import pytest

from mlx_b200 import _lib


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_results_of_another_size_or_type_are_refused(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe, libdir = str(tmp_path / "check"), os.path.dirname(_lib.LIB_PATH)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(root, "include"), os.path.join(root, "tests", "results_shim_check.cpp"), "-o", exe,
                    "-L", libdir, "-lb200q", f"-Wl,-rpath,{libdir}"], check=True, capture_output=True, text=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and "SHIM-OK" in res.stdout, res.stdout + res.stderr
