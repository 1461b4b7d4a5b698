"""Which CTA resets and writes which record of a split unit, checked on the host
(tests/paged_records_check.cpp compiles the kernels' own integer code)."""

import os
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
CUDA = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda"))


def test_records_do_not_depend_on_the_order_of_ctas(tmp_path):
    exe = tmp_path / "paged_records_check"
    subprocess.run(["g++", "-std=c++17", "-O2", f"-I{ROOT / 'cuflash-attn_b200' / 'csrc'}",
                    f"-I{CUDA / 'include'}", str(ROOT / "tests" / "paged_records_check.cpp"),
                    "-o", str(exe)], check=True)
    out = subprocess.run([str(exe), "300"], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert out.stdout.startswith("ok")
