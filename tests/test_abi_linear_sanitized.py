"""The argument checks of the bf16 products' entry points, and the rule that plans them,
under AddressSanitizer and UndefinedBehaviorSanitizer (host code)."""
import os
import subprocess
import sys

import pytest

import test_abi_sanitized as sanitized
from conftest import ROOT


def test_linear_abi_under_host_sanitizers():
    if not os.path.exists(sanitized.ASAN_LIB):
        pytest.fail(f"{sanitized.ASAN_LIB} is not built; run __graft_entry__.build()")
    if not os.path.exists(sanitized.CLANG):
        pytest.skip("clang (for its ASan runtime) is not installed")
    runtime = subprocess.run([sanitized.CLANG, "-print-file-name=libclang_rt.asan-x86_64.so"],
                             check=True, capture_output=True, text=True).stdout.strip()
    env = dict(os.environ, LD_PRELOAD=runtime, Q38M_LIB_PATH=sanitized.ASAN_LIB,
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=1", UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    source = sanitized.CHILD.replace('"test_abi.py"', '"test_abi_linear.py"').replace(
        '["-q", "-x",', '["-q", "-x", "-k", "refusals or sizes",')
    assert "test_abi_linear.py" in source and "refusals" in source
    child = subprocess.run([sys.executable, "-c", source, ROOT, sanitized.ASAN_LIB], env=env, cwd=ROOT,
                           capture_output=True, text=True, timeout=600)
    assert child.returncode == 0, child.stdout[-4000:] + child.stderr[-4000:]
    assert " passed" in child.stdout and "failed" not in child.stdout
