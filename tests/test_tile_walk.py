"""The attention tile kernels share their work by closed sums over ragged batches; the host
runs the same functions (csrc/kvm_attend_tile.cuh) against counting one by one."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_work_line_against_counting(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    exe = tmp_path / "walk"
    subprocess.run([nvcc, "-O2", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr", "-I",
                    os.path.join(ROOT, "kvmem-llama.cpp_b200", "csrc"), "-o", str(exe),
                    os.path.join(ROOT, "tests", "cpp", "tile_walk_test.cu")], check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.stdout.strip() == "ok", r.stdout
