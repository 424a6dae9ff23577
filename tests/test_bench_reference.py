"""bench.py where nibble's own CPU backend cannot be built (its sources are not there): the reference arm says so and ends well."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_reference_arm_without_the_reference():
    import oracle
    if oracle.have_ref():
        pytest.skip("nibble's CPU backend is built")
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bench.py"), "--impl", "reference"], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0, r.stderr
    line = json.loads(r.stdout)
    assert line["impl"] == "reference" and line["unavailable"]
