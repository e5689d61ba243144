"""Host-side test of the check for tensors that share memory
(csrc/overlap.hpp), built with g++ beside its driver, which compares it with
the sets of bytes of small random regions."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_overlap_against_bytes(tmp_path):
    exe = str(tmp_path / "overlap")
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(HERE, "..", "vkfft-rs_amd", "csrc"),
           os.path.join(HERE, "host", "overlap_driver.cpp"), "-o", exe]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.startswith("ok "), r.stdout[-2000:]
