"""Runs tests/ops_launch_cases.py (calls of more blocks than one launch holds) in a child process, as test_gpu_ops_torch.py does."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_calls_of_several_launches_in_a_child_process():
    env = dict(os.environ, PYTHONPATH=ROOT + os.pathsep + os.environ.get("PYTHONPATH", ""))
    env.pop("TG_HIP_RUNTIME", None)
    p = subprocess.run([sys.executable, "-u", "-m", "pytest", os.path.join(ROOT, "tests", "ops_launch_cases.py"), "-m", "gpu", "-x", "-v",
                        "-p", "no:cacheprovider"], env=env, cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert p.returncode == 0 and " passed" in p.stdout, p.stdout[-4000:] + p.stderr[-1500:]
