"""Runs tests/ops_torch_cases.py (the operators on torch tensors, their streams and captured graphs) in a child process: the main
session stays on the HIP runtime the library was built against."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_operators_on_torch_tensors_in_a_child_process():
    env = dict(os.environ, PYTHONPATH=ROOT + os.pathsep + os.environ.get("PYTHONPATH", ""))
    env.pop("TG_HIP_RUNTIME", None)
    p = subprocess.run([sys.executable, "-u", "-m", "pytest", os.path.join(ROOT, "tests", "ops_torch_cases.py"), "-m", "gpu", "-x", "-v",
                        "-p", "no:cacheprovider"], env=env, cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert p.returncode == 0 and " passed" in p.stdout, p.stdout[-4000:] + p.stderr[-1500:]
