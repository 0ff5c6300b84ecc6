"""The 8-bit KV cache on the host, from its definition (include/qwen3_hip_serve.h):
rows kept per sequence as bf16 values, blocks quantised when they are full,
attention in float64.  Test infrastructure only; nothing of the library is used."""
import numpy as np

QMAX = {"e4m3": 448.0, "int8": 127.0}
BF16_MAX = np.float32(3.38953139e38)
U = 2.0 ** -24
UB = 2.0 ** -8                      # bf16: half a step, relative


def bf16_bits(x):
    """fp32 -> bf16 bits, round to nearest even (no NaN)"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_value(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def held(x):
    """what the cache keeps of fp32 rows: finite bf16 values, as fp32"""
    x = np.where(np.isnan(x), np.float32(0), np.clip(x, -BF16_MAX, BF16_MAX)).astype(np.float32)
    return bf16_value(bf16_bits(x))


def _e4m3_table():
    t = np.zeros(256)
    for i in range(256):
        e, m = (i >> 3) & 15, i & 7
        t[i] = (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) * (-1 if i & 128 else 1)
    t[127] = t[255] = np.nan
    return t


E4M3 = _e4m3_table()


def e4m3_codes(y):
    """nearest of the 127 magnitudes, ties to the even code, beyond 448 the largest"""
    mag = E4M3[:127]
    a = np.abs(y).astype(np.float64)
    hi = np.clip(np.searchsorted(mag, a), 1, 126)
    lo = hi - 1
    mid = (mag[lo] + mag[hi]) / 2
    code = np.where((a > mid) | ((a == mid) & (hi % 2 == 0)), hi, lo)
    return (code | (np.signbit(y).astype(np.int64) << 7)).astype(np.uint8)


def quantise(x, fmt):
    """[block, dim] fp32 -> (codes uint8, scale fp32)"""
    a = np.abs(x).max().astype(np.float32)
    s = np.float32(0) if a < 2.0 ** -100 else a / np.float32(QMAX[fmt])
    if s == 0:
        return np.zeros(x.shape, np.uint8), s
    y = (x / s).astype(np.float32)
    if fmt == "e4m3":
        return e4m3_codes(y), s
    return np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8), s


def values(codes, scale, fmt):
    return (E4M3[codes] if fmt == "e4m3" else codes.view(np.int8).astype(np.float64)) * np.float64(scale)


class Sequence:
    """one sequence of one layer: rows [heads][n][dim] of K and V as the cache holds them"""

    def __init__(self, fmt, heads, dim, block):
        self.fmt, self.heads, self.dim, self.block = fmt, heads, dim, block
        self.k = np.zeros((heads, 0, dim), np.float32)
        self.v = np.zeros((heads, 0, dim), np.float32)

    def append(self, k, v):
        """k, v: fp32 [rows][heads][dim]"""
        self.k = np.concatenate([self.k, held(k).transpose(1, 0, 2)], 1)
        self.v = np.concatenate([self.v, held(v).transpose(1, 0, 2)], 1)

    def __len__(self):
        return self.k.shape[1]

    def blocks(self, which):
        """[(codes [heads][block][dim], scales [heads])] of the finished blocks"""
        x = getattr(self, which)
        out = []
        for b in range(len(self) // self.block):
            q = [quantise(x[h, b * self.block:(b + 1) * self.block], self.fmt) for h in range(self.heads)]
            out.append((np.stack([c for c, _ in q]), np.array([s for _, s in q], np.float32)))
        return out

    def read(self, which):
        """float64 [heads][n][dim] as attention sees it"""
        x = getattr(self, which).astype(np.float64)
        for b, (codes, scales) in enumerate(self.blocks(which)):
            for h in range(self.heads):
                x[h, b * self.block:(b + 1) * self.block] = values(codes[h], scales[h], self.fmt)
        return x


def attention(seq, q, pos, scale, skip=()):
    """q: float64 [rows][q_heads][dim] at positions pos ..: out and, per output, the tolerances' ingredients
    (sum p|v| / sum p, and the error a score may have, in units of U).  skip: blocks that are left out."""
    k, v = seq.read("k"), seq.read("v")
    rows, q_heads, dim = q.shape
    group = q_heads // seq.heads
    out, mean, delta = np.zeros(q.shape), np.zeros(q.shape), np.zeros((rows, q_heads, 1))
    for r in range(rows):
        keys = np.array([j for j in range(pos + r + 1) if j // seq.block not in skip], int)
        for h in range(q_heads):
            kk, vv = k[h // group, keys], v[h // group, keys]
            s = kk @ q[r, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[r, h] = p @ vv
            mean[r, h] = p @ np.abs(vv)
            delta[r, h] = score_error(np.abs(kk) @ np.abs(q[r, h]) * abs(scale), s, dim)
    return out, mean, delta


def score_error(magnitude, s, dim):
    """units of U by which a score may be off.  The dot product is 3 dim / 32 matrix instructions of 32 products each
    into an fp32 accumulator; an instruction is allowed 4 roundings of what the sum went through.  q is held to 2^-24
    (1), scale * log2 e * the page's scale is rounded three times and the product once (4), the power of two's
    argument is rounded at the score's size and the maximum's (2 |s|), and the function itself (2)."""
    return np.max((4 * 3 * dim / 32 + 5) * magnitude + 3 * np.abs(s)) + 2


def tolerance(mean, delta, ctx, bf16, out):
    """Every weight is off by delta U at most, relative, so numerator and denominator by that each; the sums of
    weights and of weights times v go through 3 x 2 matrix instructions a step of 64 keys, 4 roundings each, rescaled
    once a step, then merged (32 splits, 4 waves): a rounding each of what the sum went through, sum p|v|.  bf16:
    weights are two pieces in the numerator, the second the first's remainder rounded to bf16, and the result is
    rounded."""
    steps = ctx / 64 + 2
    rel = (2 * delta + 2 * (24 + 1) * steps + 2 * 36 + 8) * U
    tol = rel * mean
    if bf16:
        tol = tol + UB * UB * mean
        tol = tol + UB * (np.abs(out) + tol)
    return tol + 1e-37
