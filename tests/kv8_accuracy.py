"""Attention over an 8-bit cache held to fp32 accuracy: its error, as a root of the mean square over all outputs of a
call, against that of the same formula evaluated in fp32 on the host.  The worst-case tolerances of kv8_oracle.py add up
every rounding's bound and so do not see a few lost bits in all of q or of the weights; these do.  Test infrastructure
only; nothing of the library is used."""
import numpy as np

from tests import kv8_oracle as ko

# The kernel makes the host's roundings, some of them more often or larger.  A score: its factor is the product of the
# scale, log2 e and the page's scale, three roundings and the product's for the host's two (root of the sum of squares:
# 1.4).  The power of two: within an ulp where the host's exponential is within half of one (2).  The sums: 3 dim / 32
# steps of 32 products for the host's sums of dim, six times a step of 64 keys for its sums of all keys, of the same
# sizes (at most 1).  So no source is more than twice the host's; a root mean square of a few thousand values strays by
# a few percent, of the fewest here (some hundred) by a fourth: 2.5.
FACTOR = 2.5


def host(seq, q, pos, scale):
    """the formula in fp32, row by row: [rows][q_heads][dim]"""
    f = np.float32
    k, v = seq.read("k").astype(f), seq.read("v").astype(f)
    out = np.zeros(q.shape, f)
    group = q.shape[1] // seq.heads
    for r in range(q.shape[0]):
        for h in range(q.shape[1]):
            s = (k[h // group, :pos + r + 1] @ q[r, h].astype(f)) * f(scale)
            p = np.exp(s - s.max())
            out[r, h] = (p @ v[h // group, :pos + r + 1]) / p.sum(dtype=f)
    return out


def two_pieces(x):
    """x as the sum of two bf16 values, as float64: what is left of fp32 without the third"""
    first = ko.held(x.astype(np.float32))
    return first.astype(np.float64) + ko.held(x.astype(np.float32) - first)


def without_the_third_piece(seq, q, pos, scale, what):
    """the result in 64 bits but for q's, or the weights', third bf16 piece"""
    k, v = seq.read("k"), seq.read("v")
    out = np.zeros(q.shape)
    group = q.shape[1] // seq.heads
    q = two_pieces(q) if what == "q" else q.astype(np.float64)
    for r in range(q.shape[0]):
        for h in range(q.shape[1]):
            s = k[h // group, :pos + r + 1] @ q[r, h] * scale
            p = np.exp(s - s.max())
            out[r, h] = (two_pieces(p) if what == "weights" else p) @ v[h // group, :pos + r + 1] / p.sum()
    return out


class Accuracy:
    """errors gathered over the sequences of a call"""

    def __init__(self):
        self.got, self.host = 0.0, 0.0

    def add(self, seq, q, pos, scale, got):
        want = ko.attention(seq, q.astype(np.float64), pos, scale)[0]
        self.got += ((got.astype(np.float64) - want) ** 2).sum()
        self.host += ((host(seq, q, pos, scale).astype(np.float64) - want) ** 2).sum()

    def ratio(self):
        return float(np.sqrt(self.got / self.host))
