"""The C ABI's host code under AddressSanitizer and UndefinedBehaviorSanitizer,
driven through the entry points of norms between blocks and 8-bit products
(tests/sanitize_block, built by build()), as tests/test_sanitize_serving.py does for
drafted tokens and adapters."""
import os
import subprocess

import pytest

DRIVER = os.path.join(os.path.dirname(os.path.abspath(__file__)), "sanitize_block", "_build", "block_check")


def run():
    if not os.path.exists(DRIVER):
        pytest.skip("block_check is not built (build() builds it)")
    env = dict(os.environ)
    # the HIP runtime keeps allocations until the process ends: leaks are not checked
    env["ASAN_OPTIONS"] = "detect_leaks=0:abort_on_error=0:halt_on_error=1"
    env["UBSAN_OPTIONS"] = "halt_on_error=1:print_stacktrace=1"
    print("[sanitize] block_check", flush=True)
    out = subprocess.run([DRIVER], capture_output=True, text=True, timeout=300, env=env)
    assert out.returncode == 0, (out.stdout[-2000:], out.stderr[-4000:])
    assert "AddressSanitizer" not in out.stderr and "runtime error" not in out.stderr
    return out.stdout


def test_host_checks_without_gpu():
    from hachiue_amd import hip
    if hip.device_count() > 0:
        pytest.skip("a GPU is visible: the GPU test runs the full driver")
    assert "host-side checks only, 0 failed" in run()


@pytest.mark.gpu
def test_on_the_gpu():
    assert "block sanitizer run: ok" in run()
