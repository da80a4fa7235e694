"""The cut of the paged-KV attention's work, checked on the host (tests/native/kv_plan_test.cc)."""

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def test_attention_plan(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "kv_plan"
    b = subprocess.run([cxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                        f"-I{ROOT / 'pcie_pool_b200' / 'csrc'}", str(ROOT / "tests" / "native" / "kv_plan_test.cc"),
                        "-o", str(exe)], capture_output=True, text=True)
    assert b.returncode == 0, b.stderr[-4000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "kv_plan_test: ok" in r.stdout, (r.stdout + r.stderr)[-2000:]
