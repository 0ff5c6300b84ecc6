"""The recorded forward of a search, launched again by later searches with prompts in between (prompts of one row, of a
pass and of several), on the CPU against the recording stand-in for the HIP runtime (see test_host_bookkeeping_cpu):
each pointer of each recorded launch is live whenever the graph is launched, and no exec is destroyed early."""
import os
import subprocess

from tests.test_host_bookkeeping_cpu import HC, harness  # noqa: F401


def test_later_searches_replay_live_memory(harness):  # noqa: F811
    p = subprocess.run(["python3", os.path.join(HC, "drive_searches.py")], env=harness, capture_output=True, text=True,
                       timeout=900)
    print(p.stdout[-2000:])
    print(p.stderr[-4000:])
    assert p.returncode == 0, p.stderr[-4000:]
    assert "0 violations" in p.stderr and "ERROR: AddressSanitizer" not in p.stderr
