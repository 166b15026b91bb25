"""The optimizer's quotients and roots against IEEE's, over all floats."""
import subprocess

import pytest


@pytest.mark.gpu
def test_every_float(built):
    done = subprocess.run([str(built / "tests" / "gpu_pair_math")], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stdout + done.stderr
