"""What the attention kernels work out from a batch's lengths, checked on the
host by tests/kv_plan_check.cu, which includes the kernels' header: a wrong
first key would be read from outside the page table on the GPU."""
import os
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_kv_plans(tmp_path):
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    if not (Path(nvcc).exists() or shutil.which("nvcc")):
        pytest.skip("nvcc not available")
    exe = tmp_path / "kv_plan_check"
    cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O1", "-std=c++17", "--expt-relaxed-constexpr",
           "-I", str(ROOT / "include"), "-I", str(ROOT / "tier_b200" / "csrc"),
           str(ROOT / "tests" / "kv_plan_check.cu"), "-o", str(exe)]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "0 failures" in r.stdout
