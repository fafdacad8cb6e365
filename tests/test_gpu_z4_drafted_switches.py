"""Drafted sampling under the switches that choose its path, read once a process and so in child processes: with canary zones around
every buffer of the library (STATTN_DBG_REDZONE) on the row-panel kernels and, with STATTN_NO_PANELS, on the 64-column ones, where the
positions keep no projections of their states."""
import os
import re
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("panels", [True, False])
def test_drafted_sampling_touches_no_red_zone(panels):
    env = dict(os.environ, STATTN_DBG_REDZONE="1")
    env.pop("STATTN_PRECISION", None)
    if not panels:
        env["STATTN_NO_PANELS"] = "1"
    r = subprocess.run([sys.executable, "-m", "pytest", "-m", "gpu", "-x", "-q", "-p", "no:cacheprovider", "tests/test_gpu_sample_drafted.py",
                        "tests/test_gpu_sample_drafted_walk.py", "tests/test_gpu_sample_drafted_counts.py"],
                       env=env, cwd=ROOT, capture_output=True, text=True, timeout=600)
    tail = r.stdout[-3000:] + r.stderr[-1500:]
    assert r.returncode == 0, tail
    m = re.search(r"REDZONE_SCANS=(\d+)", r.stdout)
    assert m and int(m.group(1)) > 50, tail            # the scans really ran in the child
    assert re.search(r"\b\d+ passed", r.stdout) and not re.search(r"\b\d+ (failed|error)", r.stdout), tail
