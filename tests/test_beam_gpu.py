"""Beam search on the GPU: the choice of continuations against a float64 scan of all of them, and states permuted by
their parents, bit for bit."""
import ctypes

import numpy as np
import pytest

from n550_qwen3_bringup_handover_amd import abi, runtime

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def lib():
    return runtime.init()


# A row's log of the sum of exponentials: each exp within 2 U, its argument and the sums of a piece rounded (32 values a
# lane, 6 levels), the pieces joined in 64 bits: relative error of the sum, and so of its logarithm, below 64 U.  Scores
# of different rows are ordered to twice that; within a row the order is that of the logits, exactly.
LSE = 64 * U


def totals(logits, score, done, end0):
    """[W, V] scores from the definition; a finished beam has one, the rest are NaN: no continuations"""
    W, V = logits.shape
    x = np.where(np.isnan(logits), -np.inf, logits).astype(np.float64)
    total = np.full((W, V), np.nan)
    for w in range(W):
        base = float(score[w]) if np.isfinite(score[w]) else -np.inf
        if done[w]:
            total[w, end0] = base
            continue
        with np.errstate(all="ignore"):
            m = x[w].max()
            t = base + (x[w] - (m + np.log(np.exp(x[w] - m).sum())))
        total[w] = np.where(np.isnan(t), -np.inf, t)
    return total


def best(total, n):
    """the first n of [W, V] flattened: by score, then by index"""
    flat = total.reshape(-1)
    order = np.lexsort((np.arange(flat.size), -flat))          # NaN last
    return order[:n]


def run(logits, score, done, end0, end1, ld=None, offset=0, in_place=False):
    G, W, V = logits.shape
    ld = ld or V
    full = np.full((G * W, ld), 1e30, np.float32)
    full[:, :V] = logits.reshape(G * W, V)
    up = abi.DeviceBuffer.from_array
    flat = np.concatenate([np.full(offset, 1e30, np.float32), full.reshape(-1)])
    xd, sd = up(flat), up(score.astype(np.float32))
    dd = up(done.astype(np.int32))
    outs = [sd if in_place else up(np.full(G * W, 7, np.float32)), dd if in_place else up(np.full(G * W, 7, np.int32)),
            up(np.full(G * W, 7, np.int32)), up(np.full(G * W, 7, np.int32))]
    n = abi.beam_select_work(V, G, W)
    wd = up(np.full(n, 0xFF, np.uint8))
    abi.beam_select_dev(xd.ptr + 4 * offset, ld, V, G, W, sd.ptr, dd.ptr if end0 >= 0 else None, end0, end1,
                        *[o.ptr for o in outs], wd.ptr, n)          # without an end token no beam is finished
    abi.sync()
    return [o.download(t, G * W).reshape(G, W) for o, t in zip(outs, (np.float32, np.int32, np.int32, np.int32))]


def check_group(total, logits, done, end0, end1, score, fin, token, parent):
    W, V = total.shape
    want = best(total, W)
    chosen = parent.astype(np.int64) * V + token
    assert len(set(chosen.tolist())) == W and (parent >= 0).all() and (parent < W).all() and (token >= 0).all() and (token < V).all()
    flat = total.reshape(-1)
    for k in range(W):
        exact, wanted = flat[chosen[k]], flat[want[k]]
        assert not np.isnan(exact), (k, int(parent[k]), int(token[k]))
        if np.isfinite(wanted):
            assert abs(exact - wanted) <= 2 * LSE, (k, exact, wanted)
            assert abs(score[k] - exact) <= LSE + U * abs(exact) + 1e-30, (k, score[k], exact)
        else:
            assert exact == -np.inf and score[k] == -np.inf and chosen[k] == want[k], (k, chosen[k], want[k])
        assert fin[k] == int(bool(done[parent[k]]) or token[k] in (end0, end1)), k
    for w in range(W):                                          # of each beam its first continuations, in their order
        mine = token[parent == w]
        if done[w]:
            continue
        row = np.where(np.isfinite(total[w]), np.where(np.isnan(logits[w]), -np.inf, logits[w]), -np.inf)
        assert mine.tolist() == np.lexsort((np.arange(V), -row))[:len(mine)].tolist(), w


def check(logits, score, done, end0, end1, **kw):
    got = run(logits, score, done, end0, end1, **kw)
    for g in range(len(logits)):
        total = totals(logits[g], score[g], done[g], end0)
        check_group(total, logits[g], done[g], end0, end1, *[x[g] for x in got])


@pytest.mark.parametrize("G,W,V,ld,offset", [(1, 1, 1, 1, 0), (1, 4, 151936, 151936, 0), (3, 8, 5001, 5001, 0), (2, 16, 2048, 2052, 0),
                                             (2, 3, 2049, 2050, 1), (5, 2, 17, 33, 3), (1, 16, 16, 16, 0), (2, 5, 70001, 70004, 0),
                                             (7, 7, 4096, 4096, 2), (1, 16, 151936, 151936, 0),
                                             (2, 2, 300001, 300004, 0), (1, 3, 1 << 21, 1 << 21, 0), (1, 2, 1000003, 1000003, 0)])
def test_choice(G, W, V, ld, offset):
    print(f"select {G} x {W} of {V}, stride {ld}, offset {offset}", flush=True)
    rng = np.random.default_rng([G, W, V])
    logits = (rng.standard_normal((G, W, V)) * 3).astype(np.float32)
    score = -rng.uniform(0, 4, (G, W)).astype(np.float32)
    done = rng.random((G, W)) < 0.3
    done[:, 0] = False                                # someone can go on
    check(logits, score, done, V // 2, V // 3, ld=ld, offset=offset)
    check(logits, score, np.zeros_like(done), -1, -1, ld=ld, offset=offset, in_place=True)
    first = np.full((G, W), -np.inf, np.float32)
    first[:, 0] = 0
    check(logits, first, np.zeros_like(done), 0, V - 1, ld=ld, offset=offset)


def test_ties_go_to_the_lowest_index():
    V, W = 6000, 4
    logits = np.zeros((2, W, V), np.float32)
    score = np.zeros((2, W), np.float32)
    logits[1] = np.tile(np.array([1.0, 2.0, 2.0, 0.0], np.float32), V // 4)
    check(logits, score, np.zeros((2, W), bool), 3, 3)
    # the best of a row all in one lane's values, and in one wave's
    x = np.full((1, 16, V), -5.0, np.float32)
    x[0, 3, 4:4 + 16] = 9.0
    x[0, 5, 256 * np.arange(16)] = 9.0
    check(x, np.zeros((1, 16), np.float32), np.zeros((1, 16), bool), 1, 2)


def test_all_finished_and_few_left():
    rng = np.random.default_rng(5)
    W, V = 4, 300
    logits = rng.standard_normal((3, W, V)).astype(np.float32)
    score = -rng.uniform(0, 9, (3, W)).astype(np.float32)
    done = np.ones((3, W), bool)
    done[1, 2] = False
    score[2] = score[2, 0]                             # equal scores of finished beams: the lowest beam first
    check(logits, score, done, 7, 8)


def test_masked_tokens_and_rows_without_probabilities():
    rng = np.random.default_rng(6)
    W, V = 3, 5000
    logits = rng.standard_normal((6, W, V)).astype(np.float32)
    logits[0, :, 2:] = -np.inf                         # two tokens left in each row
    logits[1, 0] = -np.inf                             # a row without any
    logits[2, 1, 17] = np.nan                          # never chosen, does not count
    logits[3, 2, 4000] = np.inf                        # no probabilities: its continuations score -inf
    logits[4, 1:] = -np.inf                            # one token in all
    logits[4, 0, :] = -np.inf
    logits[4, 0, 4321] = 1.0
    logits[5] = np.nan
    check(logits, -rng.uniform(0, 1, (6, W)).astype(np.float32), np.zeros((6, W), bool), 1, -1)


def test_beams_that_are_not_in_use():
    """scores that are not finite, of running and of finished beams, and rows without probabilities, as all there is"""
    rng = np.random.default_rng(7)
    W, V = 4, 2500
    logits = rng.standard_normal((5, W, V)).astype(np.float32)
    score = np.zeros((5, W), np.float32)
    score[0] = [np.nan, -np.inf, np.inf, -1.0]
    score[1] = [np.nan, np.inf, -np.inf, np.nan]
    score[2] = -np.inf
    logits[3, :, 77] = np.inf
    logits[4] = -np.inf
    logits[4, 2, 5] = 0.0
    done = np.zeros((5, W), bool)
    done[1, 0] = done[1, 1] = done[2, 3] = True
    check(logits, score, done, 9, 9)
    check(logits, score, np.zeros((5, W), bool), -1, -1, in_place=True)


def test_select_replayed_from_a_graph(lib):
    rng = np.random.default_rng(8)
    G, W, V = 2, 4, 9000
    up = abi.DeviceBuffer.from_array
    xs = [(rng.standard_normal((G, W, V)) * 2).astype(np.float32) for _ in range(3)]
    score, done = np.zeros((G, W), np.float32), np.zeros((G, W), bool)
    xd, sd, dd = up(xs[0]), up(score), up(done.astype(np.int32))
    outs = [up(np.zeros(G * W, t)) for t in (np.float32, np.int32, np.int32, np.int32)]
    n = abi.beam_select_work(V, G, W)
    wd = abi.DeviceBuffer(n)
    call = lambda: abi.beam_select_dev(xd.ptr, V, V, G, W, sd.ptr, dd.ptr, 5, 5, *[o.ptr for o in outs], wd.ptr, n)
    call()
    runtime.check(lib.qwen3_hip_capture_begin(), "capture_begin")
    call()
    gid = ctypes.c_int(-1)
    runtime.check(lib.qwen3_hip_capture_end(ctypes.byref(gid)), "capture_end")
    try:
        for x in xs + xs:
            xd.upload(x)
            runtime.check(lib.qwen3_hip_graph_launch(gid.value), "graph_launch")
            abi.sync()
            got = [o.download(t, G * W).reshape(G, W) for o, t in zip(outs, (np.float32, np.int32, np.int32, np.int32))]
            for g in range(G):
                check_group(totals(x[g], score[g], done[g], 5), x[g], done[g], 5, 5, *[y[g] for y in got])
    finally:
        runtime.check(lib.qwen3_hip_graph_destroy(gid.value), "graph_destroy")


@pytest.mark.parametrize("G,W,slabs,runs,run,used,gap", [(1, 1, 1, 1, 16, 16, 0), (3, 4, 5, 3, 160, 96, 32), (2, 16, 2, 1, 4096, 4096, 0),
                                                        (1, 7, 3, 9, 52, 20, 4), (4, 5, 1, 2, 1028, 1028, 0), (1, 8, 56, 1, 65536, 65536, 0)])
@pytest.mark.parametrize("same", [False, True])
def test_reorder(G, W, slabs, runs, run, used, gap, same):
    """rows, runs and slabs with gaps between them that stay as they are; parents outside the group are left out"""
    rng = np.random.default_rng([G, W, slabs, runs])
    seq = runs * run + gap
    slab = G * W * seq + 2 * gap
    src = rng.integers(0, 256, slabs * slab, dtype=np.uint8)
    dst = src.copy() if same else rng.integers(0, 256, slabs * slab, dtype=np.uint8)
    parent = rng.integers(0, W, (G, W)).astype(np.int32)
    if W > 3:
        parent[0, 1], parent[-1, 2] = -1, W
    want = dst.copy()
    for s in range(slabs):
        for g in range(G):
            for w in range(W):
                p = parent[g, w]
                if 0 <= p < W:
                    for r in range(runs):
                        a, b = (s * slab + (g * W + i) * seq + r * run for i in (w, p))
                        want[a:a + used] = src[b:b + used]
    sd = abi.DeviceBuffer.from_array(src)
    dd = sd if same else abi.DeviceBuffer.from_array(dst)
    pd = abi.DeviceBuffer.from_array(parent)
    abi.beam_reorder_dev(dd.ptr, sd.ptr, pd.ptr, G, W, slabs, slab, seq, runs, run, used)
    abi.sync()
    assert np.array_equal(dd.download(np.uint8, dst.size), want)
    if not same:
        assert np.array_equal(sd.download(np.uint8, src.size), src)
