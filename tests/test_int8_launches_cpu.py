"""The launches of the 8-bit rows and products and of the rules on logits over their range of sizes, on the CPU
(tests/hostcheck/int8_launches.cpp): none is refused, and the library holds the kernels that are launched, no others."""
import os
import re
import subprocess

import pytest

from tests.test_int8_bounds_cpu import CLANG, HERE, ROOT

OBJS = [os.path.join(ROOT, "_build", o) for o in ("hip_gemm.o", "hip_model.o")]
NAMES = r"k_rows_int8|k_i8_any|k_i8_narrow|k_i8_tile|k_logits_rules"


@pytest.mark.skipif(not os.path.exists(CLANG) or not os.path.isdir(os.path.join(HERE, "hostcheck")) or
                    not all(map(os.path.exists, OBJS)), reason="no host compiler, or the library is not built here")
def test_every_kernel_is_launched(tmp_path):
    import sys
    sys.path.insert(0, os.path.join(HERE, "hostcheck"))
    import kernel_args
    # behind the harness' own macro, before the kernels
    (tmp_path / "hip_shim.h").write_text('#include_next "hip_shim.h"\n#undef hipLaunchKernelGGL\n'
                                         '#define hipLaunchKernelGGL(K, ...) launched((const void *)(K))\n')
    exe = str(tmp_path / "int8_launches")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O0", "-w", "-I", str(tmp_path), "-I",
                    os.path.join(ROOT, "n550_qwen3_bringup_handover_amd", "csrc"),
                    os.path.join(HERE, "hostcheck", "int8_launches.cpp"), "-o", exe, "-lpthread", "-ldl", "-Wl,-E"], check=True)
    p = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stdout[-600:]
    launched = set(p.stdout.split())
    built = {name for o in OBJS for name, _ in kernel_args.kernels_of(o, str(tmp_path)) if re.search(NAMES, name)}
    assert len(built) > 40
    assert built == launched, (sorted(built - launched), sorted(launched - built))
