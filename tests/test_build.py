"""The build where PyTorch is missing: the C library needs nvcc alone."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# everything counts as up to date, so nothing is compiled; an import of torch fails
WITHOUT_TORCH = """
import sys
sys.modules["torch"] = None
from sparse_ads_baselines_b200 import build
build._newer = lambda target, deps: True
print(build.build())
"""


def test_the_library_builds_without_pytorch():
    r = subprocess.run([sys.executable, "-c", WITHOUT_TORCH], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert r.stdout.strip().endswith("libtbe_b200.so")
    assert "_torch_glue.so is not built" in r.stderr  # and it says what is missing
