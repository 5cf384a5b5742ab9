"""The uneven cut of the keys by the attention of several query tokens over the 8-bit
cache (csrc/kv4_cut.h, arithmetic without device code), under
UndefinedBehaviorSanitizer: tests/sanitize/kv8_cut.cpp checks it over random batches."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_the_uneven_cut_under_sanitizers(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is not available")
    out = tmp_path / "kv8_cut"
    cmd = [gxx, "-std=c++17", "-O1", "-g", "-fsanitize=undefined",
           "-fno-sanitize-recover=undefined", "-Wall",
           str(ROOT / "tests" / "sanitize" / "kv8_cut.cpp"), "-o", str(out)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([str(out)], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0 and res.stdout.endswith("ok\n"), res.stdout + res.stderr
