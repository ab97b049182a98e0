"""Spans of a row's logits (scriptrs_amd/csrc/sfe_decode.hpp, which sfe_logits.hip takes them from), on the host."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def test_no_token_is_counted_outside_its_span(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    exe = str(tmp_path / "spans")
    subprocess.run([HIPCC, "-O2", "-std=c++17", "-x", "hip", "--cuda-host-only", "-Wno-unused-command-line-argument",
                    "-I", os.path.join(ROOT, "scriptrs_amd", "csrc"), os.path.join(ROOT, "tests", "logits_span_driver.cpp"), "-o", exe],
                   check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout + out.stderr
