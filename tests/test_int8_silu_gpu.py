"""silu(g) u of the 8-bit gated products over the whole range of g and u, on every kernel, against 64 bits.

Codes are chosen so that g and u are c_m times a scale: the scale of a column is the value itself.  Both are fp32 values that
the oracle's products give to the bit.  From there, in half steps of fp32 (2^-24), s and h being values of the exponential:

  |g| < 87   e = exp(-g) from a power of two that is off by up to 2, joined with its remainder by an fma, 1: 3, of which the
             sum takes e / (1 + e) < 1, and rounds, 1; the quotient, corrected by its remainder, 1; its product with u, 1: 6
  g <= -87   h = exp(g / 2), off by up to 2, twice; three products: 7.  1 + exp(g) is 1 to 2^-125
  g >= 87    g u: 1

so 7 in all.  h is subnormal for g < -174: what is lost is below |g| exp(g) |u| < 2^-244 |u|.  Results that are subnormal
are off by 2^-149 at most.  Where |g| < 2^-124 the quotient g / (1 + e) is subnormal, or its correction is: either rounds to
a multiple of 2^-149, by 2^-150 at most each, which u then multiplies: 2^-149 |u|.  Where silu(g) is below 2^-149 in
magnitude it is 0 as fp32, and an infinite u makes 0 times infinity, NaN, or infinity as in 64 bits.  In bf16 the remainder is not joined: the power's argument is off by (1.4427 2^-24 + 1.93e-8) |g|
and the result by ln 2 times that, 1.23 |g| 2^-24, of a quotient without its correction, 2 more; and a bf16 step."""
import numpy as np
import pytest

from n550_qwen3_bringup_handover_amd import abi, runtime
from tests import int8_oracle as io
from tests.test_int8_gpu import At, Product
from tests.test_int8_plans import SIZES

pytestmark = pytest.mark.gpu
F32 = np.float32
BIG = float(np.finfo(F32).max)


@pytest.fixture(scope="module", autouse=True)
def lib():
    return runtime.init()


def columns(rng, n, odd):
    """g and u of n columns"""
    g = rng.uniform(-200, 200, n)
    for i, (lo, hi) in enumerate(((-89, -86), (86, 89), (-105, -103), (-1, 1), (-1e-3, 1e-3), (-180, -170), (-20, 20), (-88, -86.9))):
        g[i::16] = rng.uniform(lo, hi, len(g[i::16]))
    u = rng.standard_normal(n) * 10.0 ** rng.integers(-6, 7, n)
    u[3::7] = rng.uniform(0.1, 1, len(u[3::7])) * 1e36                  # what is lost of a small silu would show
    u[5::11] = 1e-30
    if odd:
        g[8::16] = np.resize([np.inf, -np.inf, np.nan, BIG, -BIG, 1e-45, 0.0, -300.0], len(g[8::16]))
        few = np.flatnonzero(g > -150)[::13]
        u[few] = np.resize([np.inf, -np.inf, np.nan, 0.0, BIG, 1e-44], len(few))
    return g.astype(F32), u.astype(F32)


def set_values(p, rng, odd):
    p.a[:] = 0
    for b in p.b:
        b[:] = 0
    rows = np.resize(np.array([1, 1, 2, -1, 1, 3, -2], np.int8), p.m)
    p.a[:, 0], p.a[:, p.k - 1] = rows, np.resize(np.array([1, -1, 2], np.int8), p.m)
    p.b[0][:, 0] = 1
    p.b[1][:, p.k - 1] = 1
    p.sa[:] = 1
    p.sb[0][:], p.sb[1][:] = columns(rng, p.n, odd)
    p.ad = At(np.pad(p.a, ((0, 0), (0, p.lda - p.k)), constant_values=77))
    p.bd = [At(np.pad(b, ((0, 0), (0, p.ldb - p.k)), constant_values=-5)) for b in p.b]
    p.sd = [At(s) for s in [p.sa] + p.sb]


def expected(p):
    with np.errstate(all="ignore"):
        # a row at a time of each factor: the codes' products are c_m
        gf = p.a[:, :1].astype(F32) * (p.sa[:, None] * p.sb[0][None])
        uf = p.a[:, p.k - 1:].astype(F32) * (p.sa[:, None] * p.sb[1][None])
        g, u = gf.astype(np.float64), uf.astype(np.float64)
        v = g / (1 + np.exp(-g)) * u
        off = np.abs(v) * (7 * 2.0 ** -24) + np.abs(u) * 2.0 ** -244 + 2.0 ** -149
        off += np.where(np.abs(g) < 2.0 ** -124, 2.0 ** -149 * np.abs(u), 0)
        either = np.isinf(u) & (np.abs(g / (1 + np.exp(-g))) < 2.0 ** -149)
        if p.bf16:
            off += np.abs(v) * ((1.23 * np.minimum(np.abs(g), 87) + 2) * 2.0 ** -24)
            off += (np.abs(v) + off) * 2.0 ** -8 + 2.0 ** -133
    return v, off, either


def check(p):
    p.launch()
    abi.sync()
    c = p.cd.get()
    assert np.array_equal(c[:, p.n:], p.mark[:, p.n:])
    c = c[:, :p.n]
    c = io.bf16_value(c) if p.bf16 else c
    v, off, either = expected(p)
    c = c.astype(np.float64)
    with np.errstate(all="ignore"):
        over = BIG * (1 - (2.0 ** -8 if p.bf16 else 2.0 ** -24))          # may round to infinity
        good = (np.abs(c - v) <= off) | (np.isnan(c) & np.isnan(v)) | (np.isinf(c) & (np.abs(v) >= over) & (np.sign(c) == np.sign(v)))
        good |= either & np.isnan(c)
    bad = np.argwhere(~good)
    if len(bad):
        i = tuple(bad[0])
        raise AssertionError(f"{len(bad)} of {good.size}, at {i}: g {p.sb[0][i[1]]} x {p.a[i[0], 0]}, u {p.sb[1][i[1]]}: {c[i]}, {v[i]} +- {off[i]}")
    with np.errstate(all="ignore"):
        part = np.abs(c - v) / off
    print("largest part of what is allowed: %.3f" % np.max(part[np.isfinite(part)]), flush=True)


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("plan,m,n", [(s[0], s[2], s[3]) for s in SIZES if s[1]] + [("any", 70, 300)])
def test_every_kernel_over_the_whole_range(plan, m, n, bf16, odd):
    print("gated", plan, m, n, bf16, odd, flush=True)
    k = 513 if m * n < 3e6 else 129
    if plan != "any":
        assert abi.int8_plan(m, k if plan == "tile64x128-once" else 513, n, True) == plan
        k = k if plan == "tile64x128-once" else 513
    # rows of C whose pieces are whole lines, and others: their stores differ
    p = Product(m, k, n, gated=True, bf16=bf16, ldc=n + 3 if odd else -(-n // 32) * 32 + 32, **(dict(lda=k, ldb=k) if plan == "any" else {}))
    set_values(p, np.random.default_rng(m + n), odd)
    check(p)


def test_small_silus_are_not_lost():
    """g = -89 and u = 1e30: -2e-7, not 0"""
    p = Product(4, 16, 32, gated=True)
    set_values(p, np.random.default_rng(0), False)
    p.sb[0][:], p.sb[1][:] = np.linspace(-103, -87, 32), 1e30
    p.sd = [At(s) for s in [p.sa] + p.sb]
    p.a[:, 0] = 1
    p.ad = At(np.pad(p.a, ((0, 0), (0, p.lda - p.k))))
    check(p)
    assert (p.cd.get() != 0).all()
