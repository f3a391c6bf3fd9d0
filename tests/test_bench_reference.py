"""What the bench's reference arm prints where the reference's CPU library is not built."""
import json
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("config", ["1", "4"])
def test_the_reference_arm_says_when_there_is_no_reference(config):
    from oracle.oracle import REF_SO
    if os.path.exists(REF_SO):
        pytest.skip("the reference's library is built")
    r = subprocess.run([sys.executable, "bench.py", "--impl", "reference", "--config", config, "--cpu-seconds", "0.2"], cwd=ROOT,
                       stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    (line,) = [json.loads(ln) for ln in r.stdout.splitlines() if ln.startswith("{")]
    assert line["impl"] == "reference" and "not built" in line["unavailable"] and "\n" not in line["unavailable"]
    # the port's sample is called that, and nothing in the line can be taken for a rate of the reference
    assert line["kind"] == "port" and "port" in line["sample"] and "metric" not in line and "e2e" not in line and "prefill" not in line
