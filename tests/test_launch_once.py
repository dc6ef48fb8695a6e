"""The once-per-device guard around kernel attributes, on the CPU against a stand-in for the runtime."""
import os
import shutil
import subprocess

import pytest

from relay_b200 import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_a_racing_or_failed_first_call_leaves_no_launch_without_its_attribute(tmp_path):
    if shutil.which(build.host_cxx()) is None:
        pytest.skip("no host compiler")
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(build.nvcc()))), "include")
    exe = str(tmp_path / "once")
    subprocess.run([build.host_cxx(), "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "relay_b200", "csrc"),
                    "-I", cuda, "-x", "c++", os.path.join(ROOT, "tests", "cpp", "test_per_device_once.cpp"), "-o", exe, "-lpthread"],
                   check=True, timeout=300)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stderr
