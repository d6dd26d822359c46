"""The serving example over caches in 8 bits, end to end against the dense layer."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))


@pytest.mark.parametrize("flags", [
    ["--cache_dtype", "e4m3"],
    ["--cache_dtype", "e5m2", "--datatype", "fp16", "--ranks", "2", "--head_dim", "128", "--window", "50", "--sinks", "3", "--page_size", "64"],
])
def test_serving_example_validates(flags):
    cmd = [sys.executable, "-u", os.path.join(ROOT, "examples", "10_decoder_attention", "serve.py"), "--steps", "20", "-v", *flags]
    proc = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-2000:]
    assert "passed" in proc.stdout and "128 of 128 pages free" in proc.stdout
