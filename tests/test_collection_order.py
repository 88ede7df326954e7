"""The library's fresh state is looked at before any test provokes an error,
in whatever order the files are named."""
import os
import subprocess
import sys

from tests.conftest import ROOT


def test_fresh_state_first():
    files = [os.path.join("tests", f) for f in ("test_loss_lists_refusals.py", "test_adam_scalars_refusals.py",
                                                "test_abi.py")]
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", "-m", "not gpu", *files],
                       cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout[-3000:]
