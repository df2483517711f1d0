"""The example that runs the linears, the cache, attention over it and draft verification together."""
import os
import re
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_drafts_change_no_token(bits):
    r = subprocess.run([sys.executable, "-u", os.path.join(ROOT, "examples", "speculative_decode.py"), "--bits", str(bits)],
                       cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "the same tokens" in r.stdout, r.stdout + r.stderr
    steps = [int(s) for s in re.findall(r"drafts \d+: (\d+) steps", r.stdout)]
    assert steps[0] == 64 and steps[1] < 64
