"""What the 8-bit cache's store and attention read and write, on the CPU: the kernels' source compiled for the host,
every buffer against an unreadable page (tests/hostcheck/kv8_store.cpp, a thread for each of a block's, and
kv8_attend.cpp, one lane after the other).  Rows that end with a block, at its edges and in its middle, behind what
earlier calls brought or not."""
import concurrent.futures
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CLANG = "/opt/rocm/llvm/bin/clang++"


@pytest.mark.skipif(not os.path.exists(CLANG) or not os.path.isdir(os.path.join(HERE, "hostcheck")),
                    reason="no host compiler that knows the kernels' vector types")
def test_rows_and_caches_are_not_left(tmp_path):
    exe = str(tmp_path / "kv8_store")
    # unoptimised, so that every access of the source is made
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O0", "-w", "-I",
                    os.path.join(ROOT, "n550_qwen3_bringup_handover_amd", "csrc"),
                    os.path.join(HERE, "hostcheck", "kv8_store.cpp"), "-o", exe, "-lpthread"], check=True)
    p = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    assert p.returncode == 0, f"exit {p.returncode} behind\n" + p.stdout[-600:]
    assert p.stdout.endswith("every access inside, every value as defined\n")


@pytest.mark.skipif(not os.path.exists(CLANG) or not os.path.isdir(os.path.join(HERE, "hostcheck")),
                    reason="no host compiler that knows the kernels' vector types")
def test_attention_stays_in_its_buffers(tmp_path):
    """through its own launcher: single rows, turns and prompts, split keys, pages that are none, entries left out"""
    exe = str(tmp_path / "kv8_attend")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O0", "-w", "-I",
                    os.path.join(ROOT, "n550_qwen3_bringup_handover_amd", "csrc"),
                    os.path.join(HERE, "hostcheck", "kv8_attend.cpp"), "-o", exe, "-lpthread"], check=True)
    n = int(subprocess.run([exe], capture_output=True, text=True, check=True).stdout)
    def one(i):
        return subprocess.run([exe, str(i)], capture_output=True, text=True, timeout=300)
    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        for p in pool.map(one, range(n)):
            assert p.returncode == 0, f"exit {p.returncode}: {p.stdout}"
