"""The C++ classes over the matrix operators (Orthogonalizer, Muon in
include/soar_optim.hpp): they compile as C++17 and C++20 (CPU), and a program
that uses them agrees with the definition in 64 bits (GPU)."""
import subprocess
from pathlib import Path

import pytest

from test_cpp_api import _compile

SRC = Path(__file__).resolve().parent / "cpp" / "test_matrix_gpu.cpp"


@pytest.mark.parametrize("std", ["c++17", "c++20"])
def test_compiles(tmp_path, std):
    _compile(tmp_path / "t", std, SRC)


@pytest.mark.gpu
def test_matches_definition(tmp_path, cuda):
    exe = tmp_path / "t"
    _compile(exe, "c++20", SRC)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    print(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "ALL MATRIX TESTS PASSED" in r.stdout
