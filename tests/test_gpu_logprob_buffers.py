"""The decoder's buffers for log probabilities over calls of different sizes."""
import numpy as np
import pytest

import fixture_models as fm

pytestmark = pytest.mark.gpu


def test_buffers_and_graphs_stay(gpu):
    """Scores of many rows without alternatives (a larger workspace) and a
    generation of one row with 64 (larger outputs), in turn: after the first
    round nothing is made anew, and a generation without log probabilities
    keeps its graph from the start."""
    import decoder

    cfg, tensors, _ = fm.load("llama")
    dec = decoder.Decoder(cfg, tensors, max_rows=64, cache_q8=True)
    rng = np.random.default_rng(2)
    tokens, prompt = rng.integers(1, 400, 64).astype(np.int32), rng.integers(1, 400, (1, 5)).astype(np.int32)
    plain = dec.generate(prompt, 6)
    graph = dec.graphs[1, None]
    rounds = []
    for _ in range(3):
        score = dec.score(tokens)
        ids, lp = dec.generate(prompt, 6, logprobs=64)
        assert np.array_equal(ids, plain)
        if rounds:
            held, held_graphs, first_score, first_lp = rounds[0]
            assert (dec.lp, dec.lp_ws) == held and dec.graphs == held_graphs
            assert all(np.array_equal(score[k], first_score[k]) for k in score)
            assert all(np.array_equal(lp[k], first_lp[k]) for k in lp)
        rounds.append(((dec.lp, dec.lp_ws), dict(dec.graphs), score, lp))
        assert dec.graphs[1, None] is graph
        assert np.array_equal(dec.generate(prompt, 6), plain)
