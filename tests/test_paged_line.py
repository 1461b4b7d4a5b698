"""The division of work of the attention over a paged cache, checked on the
host (tests/paged_line_check.cpp compiles the kernels' own integer code)."""

import os
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
CUDA = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))


def test_line_covers_every_block_once(tmp_path):
    exe = tmp_path / "paged_line_check"
    subprocess.run(["g++", "-std=c++17", "-O2", f"-I{ROOT / 'cuflash-attn_b200' / 'csrc'}",
                    f"-I{CUDA / 'include'}", str(ROOT / "tests" / "paged_line_check.cpp"), "-o",
                    str(exe)], check=True)
    out = subprocess.run([str(exe), "1500"], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert out.stdout.startswith("ok")
