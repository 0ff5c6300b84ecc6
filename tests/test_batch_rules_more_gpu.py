"""Batches whose rules change between replayed steps, and two batches of one model under rules of their own."""
import numpy as np
import pytest

from n550_qwen3_bringup_handover_amd import model as M
from tests.test_batch_rules_gpu import MAX_SEQ, blob, plain, prompts  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [True, False])
def test_a_mask_for_each_step(plain, graph):  # noqa: F811
    """masks take a sequence's two places in turn; sequence 1's stays where it is, sequence 2's comes and goes"""
    rng = np.random.default_rng(5)
    ps = prompts(3, [7, 20], 5)
    forced = rng.integers(0, M.VOCAB, (9, 3))
    with M.Batch(plain, 3, MAX_SEQ) as b:
        b.set_graph(graph)
        b.set_rules(1, allowed=[int(forced[0, 1])])
        for s in range(3):
            b.prefill(s, ps[s])
        free = b.decode(0)[2, 0]
        seen = []
        for i, f in enumerate(forced):
            b.set_rules(0, allowed=[int(f[0])])
            if i % 3 == 0:
                b.set_rules(2, allowed=[int(f[2])], bias={int(f[2]): -5.0})
            elif i % 3 == 1:
                b.set_rules(2, bias={int(f[2]): 1e4})
            else:
                b.clear_rules(2)
            t = b.decode(1)[:, 1]
            assert t[0] == f[0] and t[1] == forced[0, 1] and (i % 3 == 2 or t[2] == f[2]), i
            seen.append(t)
    # without rules of its own a sequence's text goes on as that of a batch led along the same tokens
    with M.Batch(plain, 3, MAX_SEQ) as b:
        for s in range(3):
            b.prefill(s, ps[s])
        assert b.decode(0)[2, 0] == free
        for i, t in enumerate(seen):
            for s in range(3):
                if s != 2 or i % 3 != 2:
                    b.set_rules(s, bias={int(t[s]): 1e6})
                else:
                    b.clear_rules(s)
            assert np.array_equal(b.decode(1)[:, 1], t), i


def test_two_batches_of_one_model(plain):  # noqa: F811
    """in turn, one with the head in 8 bits, as each alone"""
    ps = prompts(4, [11, 40, 5], 6)

    def opened(which):
        b = M.Batch(plain, 2, MAX_SEQ, "fp32" if which else "e4m3")
        b.set_int8_head(which == 0)
        for s in range(2):
            b.set_rules(s, repetition=1.2 + which, presence=0.5, bias={3: 2.0 * which})
            b.prefill(s, ps[2 * which + s])
        return b

    alone = []
    for w in range(2):
        with opened(w) as b:
            alone.append(np.concatenate([b.decode(n)[:, 1:] for n in (1, 3, 4)], 1))
    a, c = opened(0), opened(1)
    got = [[], []]
    for n in (1, 3, 4):
        for w, b in enumerate((a, c)):
            got[w].append(b.decode(n)[:, 1:])
    a.close()
    c.close()
    for w in range(2):
        assert np.array_equal(np.concatenate(got[w], 1), alone[w]), w
