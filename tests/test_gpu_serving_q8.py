"""The decoder with an 8-bit cache, and its log probabilities: rope and store,
attention, log probabilities and the greedy loop together, as a server runs
them.

With float32 activations every op before and after the cache is within 2e-5 of
the reference (test_gpu_decoder.py), so the decoder is compared with the CPU
restatement of the graph whose cache is q8_ref.Cache. Where a float32
difference moves a value over a rounding border, one cached integer changes by
one: a key or value of a token by 1/127 of its block's largest, so a logit by
less than that share of the token's weight; 2e-3 of the largest logit allows a
few of them (measured differences are far below where none falls so)."""
import numpy as np
import pytest

import fixture_models as fm
import llama_ref
import q8_ref

pytestmark = pytest.mark.gpu


class RefDecoder(llama_ref.Decoder):
    """llama_ref.Decoder over 8-bit caches."""

    def __init__(self, model, **kw):
        super().__init__(model, **kw)
        c = model.c
        self.q8 = [q8_ref.Cache(c["kv_heads"], c["context"], c["head_dim"]) for _ in range(c["layers"])]

    def forward(self, tokens, positions, last_only=False):
        layer, refs = [0], self.q8
        index = np.asarray(positions)

        class Rows(list):
            """Takes the place of a layer's cache array: gathers the rows."""

            def __setitem__(self, at, row):
                self.append(row)

        self.kc, self.vc = [Rows() for _ in refs], [Rows() for _ in refs]
        plain = llama_ref.attention

        def attention(q, kc, vc, pos, kv_heads, kstart=None):
            ref = refs[layer[0]]
            ref.store(np.stack(kc), np.stack(vc), index)
            layer[0] += 1
            return q8_ref.attention(q, *ref.values(), pos)[0].astype(np.float32)

        llama_ref.attention = attention
        try:
            return super().forward(tokens, positions, last_only)
        finally:
            llama_ref.attention = plain


@pytest.mark.parametrize("name", fm.FIXTURES)
def test_steps_match_the_restatement(gpu, oracle, name):
    import decoder

    cfg, tensors, e = fm.load(name)
    dec = decoder.Decoder(cfg, tensors, a8=False, cache_q8=True, max_rows=16)
    ref = RefDecoder(llama_ref.Model(cfg, tensors), a8=False)
    P = len(e["prompt_ids"])
    want = ref.forward(e["prompt_ids"], np.arange(P))
    ok, worst, allowed = fm.near(dec.forward(e["prompt_ids"], np.arange(P)), want, 2e-3)
    assert ok, f"prompt logits: {worst} > {allowed}"
    for i, tok in enumerate(e["greedy"][:-1]):
        want = ref.forward([tok], [P + i])
        ok, worst, allowed = fm.near(dec.forward([tok], [P + i]), want, 2e-3)
        assert ok, f"step {i}: {worst} > {allowed}"


@pytest.mark.parametrize("a8", [False, True])
def test_slots_match_single_sequences(gpu, a8):
    """Three slots of a context that is not a multiple of 32: each prompt's own
    continuation, also after a slot is used again."""
    import decoder

    cfg, tensors, _ = fm.load("llama")
    cfg = dict(cfg, context=45)
    rng = np.random.default_rng(1)
    batch = decoder.Decoder(cfg, tensors, a8=a8, max_rows=32, slots=3, cache_q8=True)
    single = decoder.Decoder(cfg, tensors, a8=a8, max_rows=32, slots=1, cache_q8=True)
    for _ in range(2):
        prompts = rng.integers(1, 400, (3, 6)).astype(np.int32)
        got = batch.generate(prompts, 38)
        for i in range(3):
            assert single.generate(prompts[i:i + 1], 38)[0].tolist() == got[i].tolist(), f"slot {i}"


@pytest.mark.parametrize("q8", [False, True])
def test_generate_with_log_probabilities(gpu, q8):
    """The graph-replayed loop gives the eager loop's tokens and bits, and they
    are those of the logits."""
    import decoder

    cfg, tensors, _ = fm.load("qwen2")
    rng = np.random.default_rng(4)
    prompts = rng.integers(1, 400, (2, 5)).astype(np.int32)
    dec = decoder.Decoder(cfg, tensors, max_rows=8, slots=2, cache_q8=q8)
    ids = dec.generate(prompts, 12)
    runs = []
    for graph in (True, False, True):
        dec.reset()
        got, lp = dec.generate(prompts, 12, graph=graph, logprobs=7)
        assert np.array_equal(got, ids)
        assert np.array_equal(lp["top_ids"][..., 0], ids)  # greedy: the largest
        assert np.array_equal(lp["top_logprobs"][..., 0], lp["logprobs"])
        runs.append(lp)
    for r in runs[1:]:
        for k, v in r.items():
            assert np.array_equal(v, runs[0][k]), k
    _, none = dec.generate(prompts, 3, logprobs=0)
    assert none["top_ids"].shape == (2, 3, 0) and none["logprobs"].shape == (2, 3)
    # the last step's, from its logits
    dec.reset()
    dec.generate(prompts, 12)
    logits = dec.logits.download(np.float32, 2 * dec.vocab).reshape(2, -1)
    given, ent, top, top_lp = q8_ref.logprobs(logits, ids[:, -1], 7)
    assert np.abs(given - runs[0]["logprobs"][:, -1]).max() < 1e-5 and np.abs(ent - runs[0]["entropy"][:, -1]).max() < 1e-5
    assert np.array_equal(top, runs[0]["top_ids"][:, -1])


@pytest.mark.parametrize("cache", ["f32", "f16", "q8"])
def test_score(gpu, cache):
    """Scores in chunks of max_rows, of any slot, are those of the logits."""
    import decoder

    cfg, tensors, _ = fm.load("llama")
    kw = dict(cache_f16=cache == "f16", cache_q8=cache == "q8", slots=2)
    dec = decoder.Decoder(cfg, tensors, a8=False, max_rows=16, **kw)
    tokens = np.random.default_rng(7).integers(1, 400, 41).astype(np.int32)
    got = dec.score(tokens, top=5, slot=1)
    assert [got[k].shape for k in ("logprobs", "entropy", "top_ids", "top_logprobs")] == [(40,), (41,), (41, 5), (41, 5)]
    dec.reset()
    logits = np.concatenate([dec.forward(tokens[i:i + 16], np.arange(i, min(i + 16, 41)), np.full(min(16, 41 - i), 1))
                             for i in range(0, 41, 16)])
    given, ent, top, top_lp = q8_ref.logprobs(logits, np.append(tokens[1:], -1), 5)
    # (log probabilities here are below 20: 2^-24 (2 * 20 + 128) = 1.0e-5)
    assert np.abs(got["logprobs"] - given[:-1]).max() < 1.1e-5
    assert np.abs(got["entropy"] - ent).max() < 3e-5  # 2^-24 (128 + 128 * 3)
    assert np.array_equal(got["top_ids"], top) and np.abs(got["top_logprobs"] - top_lp).max() < 1.1e-5
    assert dec.score(tokens[:1])["logprobs"].shape == (0,)


def test_long_context(gpu):
    """Past the 8192 positions of the other caches: a prompt in chunks of whole
    blocks and in others (which requantize the block they continue) ends in
    nearly the same logits."""
    import decoder

    cfg, tensors, _ = fm.load("llama")
    cfg = dict(cfg, context=9001)
    with pytest.raises(ValueError):
        decoder.Decoder(cfg, tensors, cache_f16=True)
    tokens = np.random.default_rng(8).integers(1, 400, 9001).astype(np.int32)
    last = []
    for rows in (512, 300):
        dec = decoder.Decoder(cfg, tensors, a8=False, max_rows=rows, cache_q8=True)
        for i in range(0, 9001, rows):
            T = min(rows, 9001 - i)
            got = dec.forward(tokens[i:i + T], np.arange(i, i + T))
        last.append(got[-1])
    ok, worst, allowed = fm.near(last[0], last[1], 2e-2)
    assert ok, f"{worst} > {allowed}"


def test_refusals(gpu):
    import decoder

    cfg, tensors, _ = fm.load("llama")
    with pytest.raises(ValueError):
        decoder.Decoder(cfg, tensors, cache_f16=True, cache_q8=True)
    dec = decoder.Decoder(cfg, tensors, cache_q8=True, max_rows=4)
    for bad in (lambda: dec.score([]), lambda: dec.score([1, 2], top=65), lambda: dec.score([1, 2], top=-1),
                lambda: dec.score([1, 2], slot=1), lambda: dec.generate([[1]], 2, logprobs=65)):
        with pytest.raises(ValueError):
            bad()
    assert dec.score([1, 2, 3, 4, 5])["logprobs"].shape == (4,)  # still works
