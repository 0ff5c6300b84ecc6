"""8-bit products into rows of C that lie far apart, and of very many columns, on a machine without a GPU: what is refused,
which kernel a size goes to, and where the kernels' results land (tests/hostcheck/int8_wide.cpp)."""
import concurrent.futures
import os
import subprocess

import pytest

from n550_qwen3_bringup_handover_amd import abi, runtime
from tests.test_int8_bounds_cpu import CLANG, HERE, ROOT
from tests.test_int8_cpu import ESTATE, ETOOBIG, gated, product

no_gpu = pytest.mark.skipif(runtime.gpu_visible(), reason="accepted calls would launch")


@no_gpu
@pytest.mark.parametrize("bf16", [0, 1])
def test_more_than_four_rows_have_no_bound_on_columns(bf16):
    most = 2 ** 31 - 1
    for m in (5, 16, 33):
        for n in (1 << 27, (1 << 27) + 5, most):
            assert product(m=m, n=n, ldc=n, bf16=bf16) == ESTATE, (m, n)
            assert gated(m=m, n=n, ldh=n, bf16=bf16) == ESTATE, (m, n)
    # up to four rows: the bound that the header states
    assert product(m=4, n=(1 << 27) - 16, ldc=1 << 27) == ESTATE and product(m=4, n=1 << 27, ldc=1 << 27) == ETOOBIG


@no_gpu
@pytest.mark.parametrize("m,n", [((1 << 24) - 8 << 6, 64), ((1 << 24) - 8 << 6, 50), (5, (1 << 24) - 8 << 6), (1000, 1 << 25), (1 << 20, 65472)])
@pytest.mark.parametrize("lda", [64, 65])
def test_below_2_24_blocks_of_64_x_64_no_launch_is_too_large(m, n, lda):
    assert -(-m // 64) * -(-n // 64) <= (1 << 24) - 8
    for ld in (n, n + 5, 1 << 31):
        assert product(m=m, n=n, ldc=ld, lda=lda) == ESTATE and gated(m=m, n=n, ldh=ld, ldx=lda) == ESTATE, ld


def test_wide_rows_go_to_tiles():
    for n in (1 << 20, (1 << 20) + 16, 1 << 21):
        assert abi.int8_plan(4096, 1024, n) == "tile256", n
    # a tile's rows of C lie within 2^31 bytes as fp32
    for n in ((1 << 21) + 16, (1 << 21) + (1 << 20), 1 << 22, (1 << 22) + 16, 1 << 23):
        height = {"tile64": 64, "tile64x128": 64, "tile128": 128, "tile192x256": 192}[abi.int8_plan(4096, 1024, n)]
        assert height * n <= 1 << 29, n
    assert abi.int8_plan(4096, 1024, (1 << 23) + 16) == "narrow32"


@pytest.mark.skipif(not os.path.exists(CLANG) or not os.path.isdir(os.path.join(HERE, "hostcheck")),
                    reason="no host compiler that knows the kernels' vector types")
def test_results_in_far_rows_land_in_their_places(tmp_path):
    exe = str(tmp_path / "int8_wide")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O0", "-w", "-I",
                    os.path.join(ROOT, "n550_qwen3_bringup_handover_amd", "csrc"),
                    os.path.join(HERE, "hostcheck", "int8_wide.cpp"), "-o", exe, "-lpthread"], check=True)
    n = int(subprocess.run([exe], capture_output=True, text=True, check=True).stdout)
    def one(i):
        return subprocess.run([exe, str(i)], capture_output=True, text=True, timeout=600)
    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        for p in pool.map(one, range(n)):
            assert p.returncode == 0 and p.stdout.endswith("every result in its place\n"), f"exit {p.returncode}: {p.stdout[-400:]}"


@pytest.mark.skipif(not os.path.exists(CLANG) or not os.path.isdir(os.path.join(HERE, "hostcheck")),
                    reason="no host compiler that knows the kernels' vector types")
def test_launches_of_many_columns_cover_them_once(tmp_path):
    # behind the harness' own macro, before the kernels
    (tmp_path / "hip_shim.h").write_text('#include_next "hip_shim.h"\n#undef hipLaunchKernelGGL\n'
                                         '#define hipLaunchKernelGGL(K, GRID, BLOCK, SHM, STREAM, ...) launched(GRID, __VA_ARGS__)\n')
    exe = str(tmp_path / "int8_split")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O0", "-w", "-I", str(tmp_path), "-I",
                    os.path.join(ROOT, "n550_qwen3_bringup_handover_amd", "csrc"),
                    os.path.join(HERE, "hostcheck", "int8_split.cpp"), "-o", exe, "-lpthread"], check=True)
    p = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0 and p.stdout.endswith("every column once\n"), p.stdout
