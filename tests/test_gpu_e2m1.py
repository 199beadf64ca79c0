"""The conversions between 4-bit numbers and halves or floats, compiled into code that uses parts of a word (tests/e2m1_words_check.cu)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"


@pytest.mark.gpu
@pytest.mark.skipif(not os.path.exists(NVCC), reason="needs nvcc")
def test_every_byte_and_every_level(tmp_path):
    exe = tmp_path / "e2m1_words_check"
    r = subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "--use_fast_math", "-I", os.path.join(ROOT, "include"), "-o", str(exe),
                        os.path.join(ROOT, "tests", "e2m1_words_check.cu")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "bad=0 no error" in r.stdout, r.stdout + r.stderr
