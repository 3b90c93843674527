"""CPU tier: what `make -C vae_gan_amd/csrc` asks for and when it compiles, by make's own dry run."""
import glob
import os
import shutil
import subprocess
import sys

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vae_gan_amd", "csrc")
pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="needs make")


def dry(*args):
    r = subprocess.run(["make", "-n", "-C", CSRC, *args], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_the_library_needs_no_python_with_torch():
    out = dry("-B", "PYTHON=/no/such/python")
    assert "libvg_hip.so" in out and "torch_ops.cpp" not in out and "library alone" in out
    assert "torch_ops.cpp" not in dry("-B", "lib")
    assert "torch_ops.cpp" in dry("-B", "PYTHON=" + sys.executable)


def test_a_changed_flag_reaches_every_object():
    out = dry("-W", "Makefile", "lib")
    for src in glob.glob(os.path.join(CSRC, "*.hip")):
        name = os.path.basename(src)
        assert any("-packed-fp32-ops" in line and f"-c {name} " in line for line in out.splitlines()), name
