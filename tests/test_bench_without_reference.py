"""CPU: bench.py's reference arm where the reference's library is not built."""
from __future__ import annotations

import json
import os
import subprocess
import sys

import pytest


def test_reference_arm_says_that_it_is_unavailable():
    import oracle as om

    if os.path.exists(om.GRAPH_SO):
        pytest.skip("the reference's library is built")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "bench.py"), "--impl", "reference", "--steps", "1", "--warmup", "3"],
                       capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0, r.stderr
    line = json.loads(r.stdout.strip().splitlines()[-1])
    assert line["impl"] == "reference" and "libggml_graph.so" in line["unavailable"]
