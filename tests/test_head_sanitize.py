"""The output head's host code (checks, plans, buffer sizes) under AddressSanitizer +
UndefinedBehaviorSanitizer — CPU only: its tests of the C ABI run again, in a child
process, against the host-sanitizer build of the library."""
import os
import subprocess
import sys

import pytest

from tests.test_host_sanitize import ROOT, SAN_LIB, _asan_runtime


@pytest.mark.skipif(not SAN_LIB.exists(), reason="host-sanitizer build absent "
                    "(python mlx-recurrence_amd/build.py --host-sanitize)")
def test_output_head_host_code_under_asan_and_ubsan():
    env = dict(os.environ)
    env.update(LD_PRELOAD=str(_asan_runtime()), MLX_RECURRENCE_AMD_LIB=str(SAN_LIB),
               ASAN_OPTIONS="detect_leaks=0:abort_on_error=1", UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    res = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", "tests/test_head_api.py", "-k",
                          "abi or refus or held"], cwd=ROOT, env=env, capture_output=True, text=True, timeout=600)
    tail = (res.stdout + res.stderr)[-3000:]
    assert res.returncode == 0, tail
    assert "AddressSanitizer" not in tail and "runtime error" not in tail, tail
    assert " passed" in tail
