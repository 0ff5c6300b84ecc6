"""What the 8-bit rows, the products and the rules on logits read and write, on the CPU: the kernels' source compiled for
the host, every buffer against an unreadable page behind its end or before its start (tests/hostcheck/int8_bounds.cpp)."""
import concurrent.futures
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CLANG = "/opt/rocm/llvm/bin/clang++"


@pytest.mark.skipif(not os.path.exists(CLANG) or not os.path.isdir(os.path.join(HERE, "hostcheck")),
                    reason="no host compiler that knows the kernels' vector types")
def test_rows_products_and_rules_stay_in_their_buffers(tmp_path):
    exe = str(tmp_path / "int8_bounds")
    # unoptimised, so that every access of the source is made
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O0", "-w", "-I",
                    os.path.join(ROOT, "n550_qwen3_bringup_handover_amd", "csrc"),
                    os.path.join(HERE, "hostcheck", "int8_bounds.cpp"), "-o", exe, "-lpthread"], check=True)
    n = int(subprocess.run([exe], capture_output=True, text=True, check=True).stdout)
    def one(i):
        return subprocess.run([exe, str(i)], capture_output=True, text=True, timeout=600)
    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        for p in pool.map(one, range(n)):
            assert p.returncode == 0 and p.stdout.endswith("every access inside\n"), f"exit {p.returncode}: {p.stdout[-400:]}"
