"""Bounds of the paged-cache kernels, checked on the host
(tests/paged_bounds_check.cpp compiles the kernels' own integer code)."""

import os
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
CUDA = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))


def test_lengths_and_offsets_stay_inside_the_tables(tmp_path):
    exe = tmp_path / "paged_bounds_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fwrapv",
                    f"-I{ROOT / 'cuflash-attn_b200' / 'csrc'}", f"-I{CUDA / 'include'}",
                    str(ROOT / "tests" / "paged_bounds_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert out.stdout.startswith("ok")
