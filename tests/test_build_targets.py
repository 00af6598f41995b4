"""What `make` builds where torch is there, and where it is not."""
import os
import shutil
import subprocess
import sys

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "diffusion-model_amd", "csrc")


def planned(python, *targets):
    """The commands of a build from nothing (none of them run)."""
    if not shutil.which("make"):
        pytest.skip("no make")
    return subprocess.run(["make", "-n", "-B", "-C", CSRC, f"PYTHON={python}", *targets], capture_output=True, text=True)


def test_the_library_needs_no_torch():
    r = planned(f"{sys.executable} -S")      # (without its site-packages)
    assert r.returncode == 0 and "libisingdiff.so" in r.stdout and "idm_host.cpp" not in r.stdout, r.stderr
    assert "torch" in r.stdout + r.stderr       # says what is left out
    r = planned(f"{sys.executable} -S", "../isingdiff/_host.so")
    assert r.returncode != 0 and "torch" in r.stderr


def test_both_are_built_where_torch_is():
    r = planned(sys.executable)
    assert r.returncode == 0 and "libisingdiff.so" in r.stdout and "idm_host.cpp" in r.stdout and "/torch/include" in r.stdout, r.stderr
