"""sbamd_last_kernel and sbamd_last_splitk after the feed-forward entry points describe one and the same product
(tests/host_san/ffn_reports.cpp over the stand-in HIP runtime; no GPU)."""
import os
import shutil
import subprocess

import pytest

HOST_SAN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host_san")


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc") or shutil.which("make") is None, reason="needs hipcc and make")
def test_reports_describe_the_last_product():
    build = subprocess.run(["make", "-C", HOST_SAN, "-j8", "build/ffn_reports"], capture_output=True, text=True)
    assert build.returncode == 0, build.stdout[-3000:] + build.stderr[-3000:]
    run = subprocess.run(["make", "-C", HOST_SAN, "run-reports"], capture_output=True, text=True, timeout=300)
    out = run.stdout + run.stderr
    assert run.returncode == 0, out[-6000:]
    assert "ERROR: AddressSanitizer" not in out and "runtime error:" not in out and "LeakSanitizer" not in out, out[-6000:]
    assert "0 reports wrong" in out
