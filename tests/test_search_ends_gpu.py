"""Beams that end in the middle of a search, and greedy steps over 8-bit caches, on a model whose tokens depend on the
whole context.

The random blob's logits have a deviation of 0.64 whatever the context, so no token stands out.  With the embedding rows
of the two tokens that end a text four times as large, theirs have a deviation of 2.56: one or the other is among the
four likeliest (0.64 times 4.2 and more, among 151,936) in about a fifth of all contexts.  The contexts of one search are
much alike, so a search meets them in its first steps or not at all, and of some searches a part of the beams goes on."""
import numpy as np
import pytest

from n550_qwen3_bringup_handover_amd import model as M
from tests.test_batch_kv8_gpu import LIMIT, log_softmax, prompts

pytestmark = pytest.mark.gpu
KV = ["fp32", "e4m3", "int8"]
DEVIATION = 0.64


@pytest.fixture(scope="module")
def ending():
    b = M.qw3m_random(0x03550040, threads=16)
    off, rows, cols = M.qw3m_tensors(b)[0]
    emb = b[off:off + 2 * rows * cols].view(np.uint16).reshape(rows, cols)
    for t in M.EOS:
        row = emb[t]
        row[(row & 0x7F80) != 0] += np.uint16(2 << 7)
    with M.Model(b, max_seq=160) as m:
        yield m


def off_by(kv):
    """what a cache may do to a logit, and what launches of another kind do (see test_batch_kv8_gpu)"""
    return LIMIT.get(kv, 0.0) * DEVIATION + 6.4e-3


def until_the_end(row):
    ends = [i for i, t in enumerate(row) if t in M.EOS]
    return row[:ends[0] + 1] if ends else row, bool(ends)


@pytest.mark.parametrize("kv", KV)
def test_beams_that_end_are_padded_and_keep_their_score(ending, kv):
    """8 searches of 4 beams; prompts of 27 to 62 tokens, so that blocks of 32 fill up behind the first ends"""
    print(f"ends of beams, {kv}", flush=True)
    width, steps = 4, 14
    ps = prompts(8, [27, 29, 31, 60, 62], 11)
    with M.Batch(ending, 8 * width, 128, kv) as b:
        early, early_scores = b.beam(ps, width, 6, stop_at_eos=True)
        toks, scores = b.beam(ps, width, steps, stop_at_eos=True)
        free, _ = b.beam(ps, width, steps)
    assert np.all(np.diff(scores, axis=1) <= 0)
    ended, going, second, kept, checked, parted = set(), 0, 0, 0, 0, 0
    for g in range(8):
        before = {tuple(until_the_end(r.tolist())[0]): s for r, s in zip(early[g], early_scores[g])
                  if until_the_end(r.tolist())[1]}
        for w in range(width):
            row = toks[g, w].tolist()
            text, end = until_the_end(row)
            if end:
                ended.add(len(text) - 1)
                second += text[-1] == M.EOS[1]
                assert row[len(text):] == [M.EOS[0]] * (steps - len(text))
                if tuple(text) in before:               # ended within six steps: the same score, to the bit, after fourteen
                    kept += 1
                    assert scores[g, w] == before[tuple(text)]
            going += not end
            parted += w > 0 and not end and until_the_end(toks[g, 0].tolist())[1]
            if w not in (0, width - 1) and end:
                continue
            total, context = 0.0, ps[g]
            for t in text:
                ending.forward(context, 0)
                total += log_softmax(ending.logits())[t]
                context = np.append(context, t).astype(np.int32)
            checked += 1
            print(f"{kv} search {g} beam {w}: {len(text)} tokens, {'ended' if end else 'going on'}, {scores[g, w]:.3f} "
                  f"against {total:.3f}", flush=True)
            # tokens' errors are their own; that of a token which ends the text is four times as large
            off = off_by(kv)
            assert abs(scores[g, w] - total) <= 3 * off * np.sqrt(len(text) + (15 if end else 0)) + off
    print(f"{kv}: ends at steps {sorted(ended)}, {second} by the second token, {kept} seen earlier, {going} going on, "
          f"{checked} scores checked", flush=True)
    assert len(ended) >= 2 and max(ended) > 0, "beams have to end behind the prompt and behind a step"
    assert second >= 1 and kept >= 1 and going >= 1
    assert parted >= 1, "beams have to go on beside one that has ended"
    assert np.isin(free, M.EOS).any()                   # without the flag they go on behind it
    assert not all(r[-1] == M.EOS[0] for r in free[np.isin(free, M.EOS).any(-1)].tolist())


@pytest.mark.parametrize("kv", ["e4m3", "int8"])
def test_greedy_tokens_are_likeliest_in_their_context(ending, kv):
    """each token against a fresh fp32 forward of everything before it: within the cache's error of the largest logit.
    In another sequence's context the same tokens lie about four deviations below it, which the check has to see."""
    print(f"greedy tokens in context, {kv}", flush=True)
    ps = prompts(3, [5, 31, 70], 12)
    with M.Batch(ending, 3, 128, kv) as b:
        for s, p in enumerate(ps):
            b.prefill(s, p)
        got = np.concatenate([b.decode(20), b.decode(25)[:, 1:]], 1)     # a call repeats the token it goes on from
    assert len({tuple(g) for g in got.tolist()}) == 3
    worst, others = 0.0, []
    for s, p in enumerate(ps):
        context = p
        for i, t in enumerate(got[s].tolist()):
            ending.forward(context, 0)
            x = ending.logits().astype(np.float64)
            # two logits, each off by up to four times the deviation of such errors
            def share(t):
                scale = 4.0 if t in M.EOS or int(x.argmax()) in M.EOS else 1.0
                return (x.max() - x[t]) / (2 * 4 * scale * off_by(kv))
            worst = max(worst, share(t))
            others.append(share(int(got[(s + 1) % 3, i])))
            context = np.append(context, t).astype(np.int32)
    print(f"{kv}: largest share of the tolerance {worst:.3f}; another sequence's tokens: least {min(others):.2f}", flush=True)
    assert worst <= 1
    assert np.median(others) > 1
