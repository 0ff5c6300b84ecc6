"""Which continuations are chosen where 64 bits do not tell their scores apart, and how far the scores of rows with the
same logits may differ."""
import numpy as np
import pytest

from n550_qwen3_bringup_handover_amd import runtime
from tests.test_beam_gpu import LSE, U, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def lib():
    return runtime.init()


def test_the_largest_logits_are_taken_and_equal_scores_go_in_order():
    """logits of 1e-30 and 0 differ, their scores beside a log sum of about 9 do not"""
    V = 5000
    x = np.full((1, 2, V), -3.0, np.float32)
    x[0, 0, 4000], x[0, 0, 2500], x[0, 0, 1] = 1e-30, 0.0, -1e-30
    score = np.array([[0.0, -np.inf]], np.float32)
    got, done, token, parent = run(x, score, np.zeros((1, 2), bool), -1, -1)
    assert token.tolist() == [[2500, 4000]] and parent.tolist() == [[0, 0]]     # the two largest, by token
    assert got[0, 0] == got[0, 1] and not done.any()
    # the best alone: the largest logit, though the scores are equal
    assert run(x[:, :1], score[:, :1], np.zeros((1, 1), bool), -1, -1)[2].tolist() == [[4000]]


def test_rows_of_the_same_logits_in_another_order():
    """their log sums differ by the roundings of fp32 sums alone; each beam's tokens keep their own order"""
    rng = np.random.default_rng(21)
    V, W = 30000, 4
    row = (rng.standard_normal(V) * 2).astype(np.float32)
    x = np.stack([rng.permutation(row) for _ in range(W)])[None]
    got, _, token, parent = run(x, np.zeros((1, W), np.float32), np.zeros((1, W), bool), -1, -1)
    r = row.astype(np.float64)
    best = r.max() - (r.max() + np.log(np.exp(r - r.max()).sum()))
    assert sorted(parent[0].tolist()) == [0, 1, 2, 3]                           # every beam's best, in whatever order
    assert [int(x[0, p].argmax()) for p in parent[0]] == token[0].tolist()
    assert np.all(np.abs(got - best) <= LSE + U * abs(best)) and np.all(np.diff(got[0]) <= 0)
