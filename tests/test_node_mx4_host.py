"""The Node layer's MXFP4 calls without a GPU: tests/node/mx4_cpu.js."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_node_mx4_cpu():
    if shutil.which("node") is None:
        pytest.skip("node is not installed")
    if not os.path.exists(os.path.join(ROOT, "shared_amd", "js", "sas_napi.node")):
        pytest.skip("the addon is not built")
    p = subprocess.run(["node", os.path.join(ROOT, "tests", "node", "mx4_cpu.js")], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stdout + p.stderr
    assert len([line for line in p.stdout.splitlines() if line.startswith("ok ")]) == 3
