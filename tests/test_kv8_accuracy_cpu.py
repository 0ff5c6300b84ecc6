"""That the accuracy check of attention over 8-bit caches (kv8_accuracy.py) sees a lost bf16 piece, of q or of the
weights alone, in every kind of call that test_kv8_accuracy_gpu makes."""
import numpy as np
import pytest

from tests import kv8_accuracy as ka
from tests import kv8_oracle as ko
from tests.test_kv8_accuracy_gpu import CALLS


@pytest.mark.parametrize("what", ["q", "weights"])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,block,heads,group,counts,before", CALLS)
def test_two_pieces_are_refused(fmt, dim, block, heads, group, counts, before, what):
    rng = np.random.default_rng([dim, block, heads, group])
    acc = ka.Accuracy()
    for n, b in list(zip(counts, before))[:3]:
        n = min(n, 20)                                  # of a prompt its last rows
        s = ko.Sequence(fmt, heads, dim, block)
        s.append(*rng.standard_normal((2, b + n, heads, dim)).astype(np.float32))
        q = rng.standard_normal((n, heads * group, dim)).astype(np.float32)
        acc.add(s, q, b, 1 / np.sqrt(dim), ka.without_the_third_piece(s, q, b, 1 / np.sqrt(dim), what))
    assert acc.ratio() > ka.FACTOR, acc.ratio()


def test_the_hosts_own_fp32_passes():
    rng = np.random.default_rng(1)
    s = ko.Sequence("e4m3", 2, 64, 16)
    s.append(*rng.standard_normal((2, 100, 2, 64)).astype(np.float32))
    q = rng.standard_normal((3, 4, 64)).astype(np.float32)
    acc = ka.Accuracy()
    acc.add(s, q, 97, 0.125, ka.host(s, q, 97, 0.125))
    assert acc.ratio() == 1
