"""CPU test of the operators' workspaces: the host code over a fake of CUDA's calls."""
from __future__ import annotations

import os
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def _cuda_include():
    for home in (os.environ.get("CUDA_HOME"), "/usr/local/cuda"):
        if home and (Path(home) / "include" / "cuda_runtime_api.h").exists():
            return Path(home) / "include"
    return None


@pytest.mark.skipif(shutil.which("g++") is None or _cuda_include() is None, reason="no compiler or CUDA headers")
def test_workspaces_over_a_fake_runtime(tmp_path):
    exe = tmp_path / "operator_workspace"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{ROOT / 'include'}",
                    f"-I{ROOT / 'einsum_ir_b200' / 'csrc'}", f"-I{_cuda_include()}",
                    str(ROOT / "tests" / "operator_workspace.cpp"), "-o", str(exe), "-lpthread"], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
