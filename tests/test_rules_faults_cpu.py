"""A batch's host code while allocations, copies, launches and waits fail, each in turn, on the CPU
(tests/hostcheck/rules_faults.c): what a failed call leaves behind."""
import os
import re
import shutil
import subprocess

import pytest

from tests.test_host_bookkeeping_cpu import HC, ROOT

CSRC = os.path.join(ROOT, "n550_qwen3_bringup_handover_amd", "csrc")


@pytest.mark.skipif(not shutil.which("gcc") or not shutil.which("nm") or not os.path.isdir(HC), reason="no host compiler")
@pytest.mark.parametrize("what", ["copies", "rules"])
def test_calls_that_fail(tmp_path, what):
    flags = ["-O1", "-g", "-std=c11", "-w", "-fsanitize=address", "-fno-omit-frame-pointer",
             "-I", os.path.join(ROOT, "include"), "-I", CSRC]
    obj, exe = str(tmp_path / "faults.o"), str(tmp_path / "faults")
    subprocess.run(["gcc", *flags, "-c", os.path.join(HC, "rules_faults.c"), "-o", obj], check=True)
    names = subprocess.run(["nm", "-u", obj], check=True, capture_output=True, text=True).stdout.split()
    launches = [n for n in names if re.match(r"(qh|qm|qw3m|qwen3_hip)_", n)]
    stubs = tmp_path / "rules_faults_stubs.c"
    stubs.write_text("int fault_op(void);\n" + "".join(f"long {n}(void) {{ return fault_op() ? 5 : 0; }}\n" for n in launches))
    subprocess.run(["gcc", *flags, obj, str(stubs), "-o", exe, "-lm"], check=True)
    p = subprocess.run([exe, what], capture_output=True, text=True, timeout=600, env=dict(os.environ, ASAN_OPTIONS="detect_leaks=0"))
    print(p.stdout[-3000:])
    assert p.returncode == 0 and p.stdout.endswith("0 faults found\n"), p.stdout[:3000] + p.stderr[-3000:]
