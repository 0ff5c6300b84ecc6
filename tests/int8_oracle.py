"""What rows_int8, the 8-bit products and the rules on logits compute, in numpy, from their definitions in
include/qwen3_hip.h and include/qwen3_hip_serve.h.

Rows, sums and rules are defined step by step down to their roundings, so they are held to the bit.  The gated product's
silu is not: g and u are the products' fp32 values, and with them the kernel forms e = exp(-g), 1 + e, g / (1 + e) and
the product with u.  exp is off by at most 2 steps of fp32 (4 half steps) and reaches the sum by e / (1 + e) < 1 of it;
sum, quotient and product round once each, the quotient by up to 2.5 steps where it is not the correctly rounded one:
4 + 1 + 5 + 1 = 11 half steps of 2^-24.  exp(-g) beyond fp32's range gives 0 for g < -88.7, where the value is below
1e-36 u."""
import numpy as np

GATED = 11 * 2.0 ** -24
TINY = np.float32(2.0 ** -100)


def bf16_bits(x):
    """fp32 -> bf16 bits, ties to even; finite values"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_value(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def rows(x):
    """(codes, scales) of fp32 rows"""
    x = np.clip(np.where(np.isnan(x), np.float32(0), x), -np.finfo(np.float32).max, np.finfo(np.float32).max)
    a = np.abs(x).max(-1) if x.shape[-1] else np.zeros(x.shape[0], np.float32)
    s = np.where(a < TINY, np.float32(0), a / np.float32(127)).astype(np.float32)
    q = x / np.where(s == 0, np.float32(1), s)[:, None].astype(np.float32)
    return np.where((s == 0)[:, None], 0, np.rint(q)).astype(np.int8), s


def product(a, sa, b, sb):
    """fp32 C of codes [M][K], [N][K]"""
    acc = np.empty((a.shape[0], b.shape[0]), np.int64)
    bt = b.astype(np.float64).T                          # sums of 2^14 K < 2^53: exact
    for i in range(0, a.shape[0], 256):
        acc[i:i + 256] = (a[i:i + 256].astype(np.float64) @ bt).astype(np.int64)
    with np.errstate(over="ignore", invalid="ignore"):
        return acc.astype(np.float32) * (sa[:, None] * sb[None, :])


def gated(a, sa, g, sg, u, su):
    """64-bit silu(G) U of the products' fp32 values, and how far a result may be off"""
    gv, uv = product(a, sa, g, sg).astype(np.float64), product(a, sa, u, su).astype(np.float64)
    with np.errstate(over="ignore"):
        v = gv / (1 + np.exp(-gv)) * uv
    return v, np.abs(v) * GATED + 1e-36 * np.abs(uv)


def rules(x, vocab, token=None, n_prompt=None, n_token=None, repetition=None, presence=None, frequency=None, bias_row=None,
          bias_token=None, bias=None, n_bias=0, mask=None, mask_of=None, n_mask=0):
    out = x.copy()
    f32 = np.float32
    with np.errstate(all="ignore"):
        for i in range(x.shape[0]):
            y = out[i]
            if token is not None and 0 <= n_token[i] <= token.shape[1]:
                h = token[i, :n_token[i]]
                from_ = min(max(n_prompt[i] if n_prompt is not None else 0, 0), len(h))
                ok = (h >= 0) & (h < vocab)
                seen = np.unique(h[ok])
                if repetition is not None:
                    r = f32(repetition[i])
                    y[seen] = np.where(y[seen] > 0, y[seen] / r, y[seen] * r)
                v, c = np.unique(h[from_:][ok[from_:]], return_counts=True)
                if frequency is not None:
                    y[v] = y[v] - f32(frequency[i]) * c.astype(f32)
                if presence is not None:
                    y[v] = y[v] - f32(presence[i])
            if bias_row is not None and bias_row[i] >= 0 and bias_row[i + 1] <= n_bias:
                last = {int(bias_token[j]): j for j in range(bias_row[i], bias_row[i + 1])}
                for v, j in last.items():
                    if 0 <= v < vocab:
                        y[v] = y[v] + f32(bias[j])
            if mask is not None:
                m = i if mask_of is None else mask_of[i]
                if 0 <= m < n_mask:
                    bits = np.unpackbits(np.ascontiguousarray(mask[m]).view(np.uint8), bitorder="little")[:vocab]
                    y[bits == 0] = -np.inf
    return out
