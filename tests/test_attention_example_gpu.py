"""The serving example end to end: prompts, single tokens, pages taken and given back, against the dense layer."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))


@pytest.mark.parametrize("flags", [
    [],
    ["--datatype", "fp16", "--ranks", "2", "--head_dim", "128", "--window", "50", "--sinks", "3", "--page_size", "32"],
    ["--ranks", "1", "--heads", "5", "--key_heads", "1", "--hidden", "320", "--page_size", "8", "--prompts", "3", "200"],
])
def test_serving_example_validates(flags):
    cmd = [sys.executable, "-u", os.path.join(ROOT, "examples", "10_decoder_attention", "serve.py"), "--steps", "3", "-v", *flags]
    proc = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-2000:]
    assert "passed" in proc.stdout and "128 of 128 pages free" in proc.stdout
