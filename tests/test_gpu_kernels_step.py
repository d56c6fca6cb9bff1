"""The local operators and the collectives together, as a training step of two ranks uses them (one process of its own)."""
import os
import subprocess
import sys

import pytest


@pytest.mark.gpu
def test_training_step_of_two_ranks():
    child = os.path.join(os.path.dirname(os.path.abspath(__file__)), "shard_step_child.py")
    r = subprocess.run([sys.executable, child], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "sharded step ok" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
