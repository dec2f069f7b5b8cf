"""Beam search over the paged cache (lrq_beam_*) against a search that scores
every continuation with the oracle's single-stream logits."""
import math

import numpy as np
import pytest

from helpers import build_pair
from lrrt_b200 import native as N
from lrrt_b200 import qwen as Q
from lrrt_b200 import synthetic as S

pytestmark = pytest.mark.gpu

# A logit's relative error is at most 1e-4 (as everywhere in these tests); a
# log-probability is a difference of two of them, a score a sum of `steps`.
LOGIT_RTOL = 1.0e-4


def oracle_logits(oracle, tokens):
    """The logits after `tokens`, from an empty cache."""
    for cache in oracle.key_cache + oracle.value_cache:
        cache[:] = 0
    for i, token in enumerate(tokens):
        oracle.decode(oracle.embedding(int(token)), i, 1)
    return oracle.logits.astype(np.float64).copy()


def oracle_search(oracle, prompt, beams, steps, eos=None):
    """[(score, tokens)], best first, and the smallest gap between a score that
    was kept and the next one."""
    found, gap, size = [(0.0, [])], math.inf, 0.0
    for _ in range(steps):
        every = []
        for k, (score, tokens) in enumerate(found):
            if eos is not None and eos in tokens:
                every.append((-score, k, eos, tokens + [eos]))
                continue
            x = oracle_logits(oracle, list(prompt) + tokens)
            size = max(size, np.abs(x).max())
            log_p = x - (x.max() + np.log(np.exp(x - x.max()).sum()))
            for t in np.argsort(-log_p, kind="stable")[:beams + 1]:
                every.append((-(score + log_p[t]), k, int(t), tokens + [int(t)]))
        every.sort(key=lambda c: c[:3])
        gaps = np.diff([c[0] for c in every[:beams + 1]])
        gap = min([gap, *gaps])
        found = [(-c[0], c[3]) for c in every[:beams]]
    return found, gap, size


@pytest.mark.parametrize("page_size,eos", [(16, None), (1, None), (7, "found"), (64, None)])
def test_beam_search_matches_the_oracle(gpu, page_size, eos):
    layers, vocab, beams, steps = 2, 512, 3, 5
    model, oracle, _, _ = build_pair(seed=41, layers=layers, vocab=vocab, capacity=96,
                                     max_tokens=8)
    model.enable_prefill(64)
    prompts = [S.prompt(400 + i, n, vocab) for i, n in enumerate((17, 1, 32, 6))]
    token = Q.NO_TOKEN
    if eos:  # a token that the best continuation of the first prompt meets on its way
        token = oracle_search(oracle, prompts[0], beams, steps)[0][0][1][1]
    with Q.Beam(model, len(prompts), beams, 96, page_size, token) as search:
        tokens, scores = search.search(prompts, steps)
        again, again_scores = search.search(prompts, steps)  # the captured step, from the start
        assert np.array_equal(tokens, again) and np.array_equal(scores, again_scores)
    for g, prompt in enumerate(prompts):
        want, gap, size = oracle_search(oracle, prompt, beams, steps,
                                        None if token == Q.NO_TOKEN else token)
        bound = 2 * steps * LOGIT_RTOL * max(1.0, size)
        assert np.abs(scores[g] - [s for s, _ in want]).max() <= bound, g
        # The order is the oracle's unless it hangs on less than the scores' error.
        assert gap > 0
        if gap > 2 * bound:
            assert tokens[g].tolist() == [t for _, t in want], g
    model.close()


def test_one_beam_is_greedy(gpu):
    """With one beam the search is greedy decoding; 40 groups run the wide GEMMs."""
    layers, vocab, steps = 2, 4096, 12
    model, oracle, _, _ = build_pair(seed=43, layers=layers, vocab=vocab, capacity=96,
                                     max_tokens=steps)
    model.enable_prefill(64)
    prompts = [S.prompt(500 + i, 1 + i, vocab) for i in range(40)]
    with Q.Beam(model, len(prompts), 1, 80) as search:
        tokens, _ = search.search(prompts, steps)
    with Q.Batch(model, len(prompts), 80, steps) as batch:
        for stream, prompt in enumerate(prompts):
            batch.prefill(stream, prompt)
        greedy, _ = batch.decode(steps)
    assert np.array_equal(tokens[:, 0], greedy)
    model.close()


def test_many_beams(gpu):
    """Half of a small vocabulary as beams, one page after another filled."""
    model, oracle, _, _ = build_pair(seed=44, layers=1, vocab=64, capacity=32, max_tokens=4)
    model.enable_prefill(32)
    with Q.Beam(model, 1, 32, 32, 4, 5) as search:
        tokens, scores = search.search([[3, 9]], 2)
    assert (np.diff(scores[0]) <= 0).all()
    assert len({tuple(t) for t in tokens[0].tolist()}) == 32
    want, _, size = oracle_search(oracle, [3, 9], 32, 2, 5)
    bound = 4 * LOGIT_RTOL * max(1.0, size)
    assert np.abs(scores[0] - [s for s, _ in want]).max() <= bound
    model.close()


def test_beam_search_refuses(gpu):
    model, _, _, _ = build_pair(seed=45, layers=1, vocab=64, capacity=32, max_tokens=4)
    with pytest.raises(N.LrrtError, match="not enabled"):
        Q.Beam(model, 1, 2, 32)
    model.enable_prefill(16)
    for arguments in ((0, 2, 32), (1, 33, 32), (9, 2, 32), (1, 2, 33), (1, 2, 0)):
        with pytest.raises(N.LrrtError, match="beam search needs"):
            Q.Beam(model, *arguments)
    with Q.Beam(model, 2, 2, 16) as search:
        for prompts, steps, text in (([[1], []], 2, "empty"), ([[1] * 15, [1]], 3, "capacity"),
                                     ([[1], [64]], 2, "out of range"), ([[1], [2]], 0, "step")):
            with pytest.raises(N.LrrtError, match=text):
                search.search(prompts, steps)
        with pytest.raises(ValueError, match="prompts"):
            search.search([[1]], 2)
        with pytest.raises(N.LrrtError, match="beam searches"):
            model.enable_prefill(16)
        search.search([[1] * 14, [1]], 3)
    model.close()
