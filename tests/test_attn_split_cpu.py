"""How the packed attention's work is split, compiled for the host
(tests/cpp/test_attn_split.cu)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")


@pytest.mark.skipif(not (os.path.exists(NVCC) or shutil.which(NVCC)), reason="needs nvcc")
def test_units_of_tiles_against_loops(tmp_path):
    exe = tmp_path / "test_attn_split"
    r = subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", "--expt-relaxed-constexpr",
                        "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "project-aaedn_b200", "csrc"),
                        "-I", os.path.join(ROOT, "project-aaedn_b200", "host"),
                        os.path.join(ROOT, "tests", "cpp", "test_attn_split.cu"), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "PASSED" in r.stdout, r.stdout + r.stderr
