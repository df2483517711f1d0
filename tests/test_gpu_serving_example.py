"""The example that runs pages and slots, adapters, rotary positions, attention and sampling together, with requests that come
and go: every request's tokens are those that it gets alone."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("bits,requests,rows", [(16, 7, 3), (8, 9, 4), (4, 6, 20)])
def test_requests_get_the_tokens_they_get_alone(bits, requests, rows):
    r = subprocess.run([sys.executable, "-u", os.path.join(ROOT, "examples", "batched_serving.py"), "--bits", str(bits),
                        "--requests", str(requests), "--rows", str(rows)], cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "the same tokens alone" in r.stdout, r.stdout + r.stderr
