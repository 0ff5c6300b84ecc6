"""Rows as int8 codes and products of such codes on the GPU, against their definitions (tests/int8_oracle.py).  Padding
between rows holds arbitrary codes where a call may read it, and is compared afterwards where it may not write."""
import numpy as np
import pytest

from n550_qwen3_bringup_handover_amd import abi, runtime
from tests import int8_oracle as io

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module", autouse=True)
def lib():
    return runtime.init()


class At:
    """an array on the device, `shift` bytes behind a 256-byte aligned address"""

    def __init__(self, x, shift=0):
        x = np.ascontiguousarray(x)
        self.buf = abi.DeviceBuffer.from_array(np.concatenate([np.zeros(shift, np.uint8), x.reshape(-1).view(np.uint8)]))
        self.ptr, self.shape, self.dtype, self.shift = self.buf.ptr + shift, x.shape, x.dtype, shift

    def get(self):
        raw = self.buf.download(np.uint8, self.shift + int(np.prod(self.shape)) * self.dtype.itemsize)
        return raw[self.shift:].copy().view(self.dtype).reshape(self.shape)


def padded(rng, x, ld, dtype=np.int8):
    full = rng.integers(-128, 128, (x.shape[0], ld)).astype(dtype)
    full[:, :x.shape[1]] = x
    return full


def quantise(x, bf16=False, ldx=None, ldq=None, shift_x=0, shift_q=0):
    rows, k = x.shape
    ldx, ldq = ldx or max(k, 1), ldq or max(k, 1)
    full = np.full((rows, ldx), np.nan, F32)
    full[:, :k] = x
    xd = At((full.view(np.uint32) >> 16).astype(np.uint16) if bf16 else full, shift_x)
    qd, sd = At(np.full((rows, ldq), 77, np.int8), shift_q), At(np.full(rows, np.nan, F32))
    abi.rows_int8_dev(qd.ptr, ldq, sd.ptr, xd.ptr, ldx, bf16, rows, k)
    abi.sync()
    q = qd.get()
    assert (q[:, k:] == 77).all()
    return q[:, :k], sd.get()


ROWS = [(1, 1024), (3, 1), (1, 5), (7, 64), (5, 100), (2, 255), (9, 1001), (64, 2048), (2, 4096), (3, 5000), (2, 8192), (1, 12289),
        (2, 20000), (1, 131071), (1500, 640), (1025, 256), (1030, 77), (4, 512), (1026, 1024), (1027, 2048), (4096, 1025), (4097, 2047),
        (256, 8192), (257, 8191), (300, 4097)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,k", ROWS)
def test_rows(rows, k, bf16):
    print("rows", rows, k, bf16, flush=True)
    rng = np.random.default_rng(rows * 1000 + k)
    x = rng.standard_normal((rows, k)).astype(F32) * F32(10.0) ** rng.integers(-6, 7, (rows, 1)).astype(F32)
    if bf16:
        x = io.bf16_value(io.bf16_bits(x))
    want_q, want_s = io.rows(x)
    for ldx, ldq, sx, sq in ((None, None, 0, 0), (-(-k // 8) * 8 + 8, -(-k // 16) * 16 + 16, 0, 0), (k + 3, k + 5, 4, 1)):
        q, s = quantise(x, bf16, ldx, ldq, sx, sq)
        assert np.array_equal(s, want_s) and np.array_equal(q, want_q)


@pytest.mark.parametrize("bf16", [False, True])
def test_rows_at_the_borders_of_their_codes(bf16):
    """quotients next to n + 1/2, where a quotient that is one step off would round to the other code"""
    rng = np.random.default_rng(5)
    x = np.empty((64, 2048), F32)
    for r in range(64):
        a = F32(rng.uniform(1, 2) * 2.0 ** rng.integers(-90, 100))
        if bf16:
            a = io.bf16_value(io.bf16_bits(np.array([a])))[0]
        s = a / F32(127)
        n = rng.integers(-126, 126, 2048) + 0.5
        y = (n * float(s)).astype(F32)
        bits = y.view(np.int32) + rng.integers(-2, 3, 2048).astype(np.int32)
        x[r] = np.clip(bits.view(F32), -a, a)
        x[r, 7] = -a
    if bf16:
        x = io.bf16_value(io.bf16_bits(x))
    q, s = quantise(x, bf16)
    want_q, want_s = io.rows(x)
    assert np.array_equal(s, want_s) and np.array_equal(q, want_q)


def test_rows_of_odd_values():
    big = np.finfo(F32).max
    x = np.zeros((9, 300), F32)
    x[1] = np.nan
    x[2, 5], x[2, 6], x[2, 7] = np.inf, -np.inf, 1.0
    x[3, :3] = [np.nan, 2.0, -1.0]
    x[4] = 2.0 ** -101                         # below the smallest scale
    x[5] = 2.0 ** -100
    x[6, 0], x[6, 1] = big, -big / 2
    x[7] = 1e-44                               # subnormal
    x[8] = -3.0
    q, s = quantise(x)
    want_q, want_s = io.rows(x)
    assert np.array_equal(s, want_s) and np.array_equal(q, want_q)
    assert s[0] == s[1] == s[4] == s[7] == 0 and not q[[0, 1, 4, 7]].any()
    assert q[2, 5] == 127 and q[2, 6] == -127 and (q[8] == -127).all() and (q[5] == 127).all()


def test_bf16_rows_of_odd_values():
    x = np.zeros((4, 200), F32)
    x[0, :4] = [np.inf, -np.inf, np.nan, 3e38]
    x[1] = np.nan
    x[2, :3] = [1.0, np.nan, -2.0]
    x[3] = io.bf16_value(np.array([1], np.uint16))[0]            # the smallest subnormal
    q, s = quantise(x, True)
    want_q, want_s = io.rows(x)
    assert np.array_equal(s, want_s) and np.array_equal(q, want_q) and s[1] == s[3] == 0


@pytest.mark.parametrize("rows,k,bf16", [(9000, 1001, False), (70000, 130, False), (2300, 4000, False), (1100, 8191, False),
                                         (700, 13000, False), (17000, 1000, True), (4200, 4096, True)])
def test_more_rows_than_the_caches_hold(rows, k, bf16):
    """rows of other strides, too: those that are read past the caches, and those that are not aligned for it"""
    print("rows", rows, k, bf16, flush=True)
    x = np.random.default_rng(k).standard_normal((rows, k), dtype=F32)
    if bf16:
        x = io.bf16_value(io.bf16_bits(x))
    want_q, want_s = io.rows(x)
    for ldx in (-(-k // 8) * 8, k):
        q, s = quantise(x, bf16, ldx, -(-k // 8) * 8 + 8)
        assert np.array_equal(s, want_s) and np.array_equal(q, want_q)


def test_no_rows_and_rows_of_nothing():
    abi.rows_int8_dev(None, 0, None, None, 0, False, 0, 0)
    sd = At(np.full(3, np.nan, F32))
    abi.rows_int8_dev(None, 0, sd.ptr, None, 0, True, 3, 0)
    abi.sync()
    assert (sd.get() == 0).all()


class Product:
    def __init__(self, m, k, n, gated=False, bf16=False, lda=None, ldb=None, ldc=None, shift=0, seed=0, full=False):
        rng = np.random.default_rng(seed * 7919 + m * 31 + k * 17 + n)
        lo = -128 if full else -127
        draw = lambda r: rng.integers(lo, 128, (r, k)).astype(np.int8)      # noqa: E731
        up = -(-k // 16) * 16
        self.m, self.k, self.n, self.bf16, self.gated = m, k, n, bf16, gated
        self.lda, self.ldb, self.ldc = lda or max(up, 16), ldb or max(up, 16), ldc or n
        self.a, self.b = draw(m), [draw(n) for _ in range(1 + gated)]
        self.sa = rng.uniform(0.5, 1.5, m).astype(F32) / F32(100)
        self.sb = [rng.uniform(0.5, 1.5, n).astype(F32) / F32(20 * max(k, 1) ** 0.5) for _ in range(1 + gated)]
        self.ad = At(padded(rng, self.a, self.lda), shift)
        self.bd = [At(padded(rng, b, self.ldb), shift) for b in self.b]
        self.sd = [At(s) for s in [self.sa] + self.sb]
        self.mark = np.full((m, self.ldc), 0x7FC1 if bf16 else 7.25, np.uint16 if bf16 else F32)
        self.cd = At(self.mark)

    def launch(self):
        s = [x.ptr for x in self.sd]
        if self.gated:
            abi.gemm_int8_gate_up_silu_dev(self.cd.ptr, self.ldc, self.bf16, self.ad.ptr, self.lda, s[0], self.bd[0].ptr, s[1],
                                           self.bd[1].ptr, s[2], self.ldb, self.m, self.k, self.n)
        else:
            abi.gemm_int8_dev(self.cd.ptr, self.ldc, self.bf16, self.ad.ptr, self.lda, s[0], self.bd[0].ptr, self.ldb, s[1],
                              self.m, self.k, self.n)

    def check(self):
        abi.sync()
        c = self.cd.get()
        assert np.array_equal(c[:, self.n:], self.mark[:, self.n:])
        c = c[:, :self.n]
        if not self.gated:
            want = io.product(self.a, self.sa, self.b[0], self.sb[0])
            want = io.bf16_bits(want) if self.bf16 else want
            bad = np.argwhere(c != want)
            assert not len(bad), (len(bad), bad[:4], c[tuple(bad[0])], want[tuple(bad[0])])
            return
        want, off = io.gated(self.a, self.sa, self.b[0], self.sb[0], self.b[1], self.sb[1])
        if self.bf16:                                   # and a rounding to bf16
            c, off = io.bf16_value(c), off + (np.abs(want) + off) * 2.0 ** -8
        assert (np.abs(c - want) <= off).all(), np.max(np.abs(c - want) / off)

    def run(self):
        print("product", self.m, self.k, self.n, "gated" * self.gated, "bf16" * self.bf16, self.lda, self.ldb, self.ldc, flush=True)
        self.launch()
        self.check()


SHAPES = [(1, 1, 1), (1, 16, 16), (1, 64, 17), (1, 1024, 4096), (1, 1000, 333), (2, 129, 40), (3, 4096, 64), (7, 200, 1000),
          (15, 2048, 96), (16, 1024, 4096), (16, 1023, 520), (17, 1024, 320), (31, 65, 200), (33, 2048, 1024), (48, 1024, 777),
          (64, 1024, 2816), (64, 8192, 48), (64, 2000, 1024), (65, 512, 130), (100, 1024, 512), (127, 333, 257), (128, 1024, 4096),
          (129, 640, 128), (200, 2048, 1024), (255, 144, 2500), (257, 1024, 769), (333, 1001, 2501), (512, 2048, 1024),
          (700, 100, 3000), (1024, 1024, 1024), (1500, 2048, 384), (2048, 512, 1500), (3000, 96, 48), (600, 40, 9000), (2300, 1100, 2050)]


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_products(m, k, n):
    Product(m, k, n).run()


@pytest.mark.parametrize("m,k,n", SHAPES[::3] + [(1, 2048, 151936), (5, 1024, 30000), (64, 1024, 40000), (40, 1500, 20001)])
def test_products_as_bf16_and_wide_ones(m, k, n):
    Product(m, k, n, bf16=True, seed=1).run()
    if n > 9000:
        Product(m, k, n, seed=2).run()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("m,k,n", [(1, 1024, 2816), (1, 33, 5), (4, 1024, 1000), (16, 512, 48), (30, 1001, 300), (64, 1024, 2816),
                                   (64, 96, 30000), (90, 300, 200), (128, 1024, 640), (300, 1024, 1000), (1000, 512, 2000), (1999, 1024, 700)])
def test_gated_products(m, k, n, bf16):
    Product(m, k, n, gated=True, bf16=bf16, seed=3).run()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,k,n", [(1, 1000, 100), (20, 300, 70), (64, 1024, 256), (130, 513, 140), (520, 777, 600)])
@pytest.mark.parametrize("how", ["tight", "odd strides", "odd addresses", "wide strides", "a alone", "b alone"])
def test_strides_and_alignments(m, k, n, gated, how):
    up = -(-k // 16) * 16
    kw = {"tight": dict(lda=k, ldb=k), "odd strides": dict(lda=k + 1, ldb=k + 7), "odd addresses": dict(shift=3),
          "wide strides": dict(lda=up + 48, ldb=up + 4096), "a alone": dict(lda=up + 16, ldb=up + 4),
          "b alone": dict(lda=up + 2, ldb=up)}[how]
    Product(m, k, n, gated=gated, ldc=n + 5, seed=4, **kw).run()


def test_largest_sums():
    """every product 2^14 or -2^14 + 2^7, up to the longest K: sums up to 2^31 - 2^14"""
    for m, k, n in ((2, 131071, 33), (70, 131071, 70), (200, 131072 - 64, 130), (16, 131071, 40000)):
        p = Product(m, k, n, full=True)
        p.a[:] = -128
        p.b[0][:] = -128
        p.b[0][n // 2:] = 127
        p.ad, p.bd = At(padded(np.random.default_rng(0), p.a, p.lda)), [At(padded(np.random.default_rng(0), p.b[0], p.ldb))]
        p.run()


def test_codes_of_all_values():
    for m, k, n in ((1, 1024, 300), (50, 700, 300), (300, 1024, 300)):
        Product(m, k, n, full=True, seed=5).run()


def test_scales_that_are_not_numbers_stay_in_their_rows():
    p = Product(40, 256, 50)
    p.sa[3], p.sa[5], p.sb[0][7] = np.nan, np.inf, -np.inf
    p.sd = [At(s) for s in [p.sa] + p.sb]
    p.launch()
    abi.sync()
    with np.errstate(all="ignore"):
        want = io.product(p.a, p.sa, p.b[0], p.sb[0])
    assert np.array_equal(p.cd.get(), want, equal_nan=True)


def test_nothing_to_multiply():
    abi.gemm_int8_dev(None, 4, False, None, 16, None, None, 16, None, 0, 16, 4)
    abi.gemm_int8_dev(None, 0, False, None, 16, None, None, 16, None, 4, 16, 0)
    for gated in (False, True):
        p = Product(3, 0, 5, gated=gated)
        p.launch()
        abi.sync()
        assert (p.cd.get() == 0).all()


@pytest.mark.parametrize("m,k,n", [(1, 1024, 4096), (64, 1024, 4096), (200, 1024, 512), (600, 512, 640)])
def test_two_calls_give_the_same_bits_and_a_graph_too(m, k, n):
    """recorded once with the rows' quantisation before it, replayed over changing rows with other calls between"""
    L = runtime.lib()
    rng = np.random.default_rng(9)
    p, other = Product(m, k, n, gated=True), Product(33, 300, 70)
    x = At(np.zeros((m, k), F32))

    def step():
        abi.rows_int8_dev(p.ad.ptr, p.lda, p.sd[0].ptr, x.ptr, k, False, m, k)
        p.launch()
        abi.gemm_int8_dev(p.cd2.ptr, n, True, p.ad.ptr, p.lda, p.sd[0].ptr, p.bd[1].ptr, p.ldb, p.sd[2].ptr, m, k, n)

    import ctypes
    p.cd2 = At(np.zeros((m, n), np.uint16))
    g = ctypes.c_int()
    runtime.check(L.qwen3_hip_capture_begin())
    step()
    runtime.check(L.qwen3_hip_capture_end(ctypes.byref(g)))
    for _ in range(4):
        x.buf.upload(rng.standard_normal((m, k)).astype(F32))
        step()
        abi.sync()
        eager = [p.cd.get(), p.cd2.get()]
        other.run()
        p.cd.buf.upload(p.mark)
        runtime.check(L.qwen3_hip_graph_launch(g.value))
        abi.sync()
        assert np.array_equal(eager[0], p.cd.get()) and np.array_equal(eager[1], p.cd2.get())
        p.a, p.sa = p.ad.get()[:, :k], p.sd[0].get()
        p.check()
    runtime.check(L.qwen3_hip_graph_destroy(g.value))
