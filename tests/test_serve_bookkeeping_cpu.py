"""Host bookkeeping of batches with 8-bit caches and of beam search (graphs of the step and of the search's forward,
workspaces, closing order), on the CPU against the recording stand-in for the HIP runtime (see
test_host_bookkeeping_cpu)."""
import os
import subprocess

from tests.test_host_bookkeeping_cpu import HC, harness  # noqa: F401


def test_serving_calls_are_clean(harness):  # noqa: F811
    p = subprocess.run(["python3", os.path.join(HC, "drive_serve.py")], env=harness, capture_output=True, text=True,
                       timeout=900)
    print(p.stdout[-2000:])
    print(p.stderr[-4000:])
    assert p.returncode == 0, p.stderr[-4000:]
    assert "0 violations" in p.stderr and "ERROR: AddressSanitizer" not in p.stderr
