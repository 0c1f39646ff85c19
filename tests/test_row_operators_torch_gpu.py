"""The row operators on the torch provider (a process of its own): streams, captured graphs."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


def test_streams_and_graphs_of_torch():
    env = dict(os.environ, DPNP_AMD_MEMORY="torch")
    env.pop("DPNP_AMD_BLOCK_TORCH", None)
    r = subprocess.run([sys.executable, "-u", os.path.join(HERE, "row_operators_torch_check.py")], env=env, text=True,
                       capture_output=True, timeout=110)
    assert r.returncode == 0 and r.stdout.rstrip().endswith("OK"), (r.returncode, r.stdout[-1500:], r.stderr[-3000:])
