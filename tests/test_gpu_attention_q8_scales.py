"""Attention over the 8-bit cache with scales far from one: its weights hold the
value scales, its scores' factor the key scales and the query's exponent."""
import numpy as np
import pytest

import attention_bound
import test_gpu_cache_q8 as cache_tests

pytestmark = pytest.mark.gpu
rt = cache_tests.rt


@pytest.mark.parametrize("T,room", [(1, None), (3, 1 << 18), (128, 1 << 18)])
@pytest.mark.parametrize("near", [-90, -64, -30, 0, 30, 64, 100])
def test_value_scales(gpu, rt, T, room, near):
    """Equal scores, so an output is the mean of the values, of two blocks whose
    scales are around 2^near. A weight's error: the logarithm of its scale's
    fraction, 2^-23, the offset, of magnitude 8 to 16, 2^-21, together times
    ln 2; the exponential, one unit in the last place, 2^-23; two parts, 2^-22. In the
    sum of weights the scale's reciprocal, 2^-23 twice. Sums and the division: five
    roundings of 2^-24. (2^-23 + 2^-21) ln 2 + 3 * 2^-23 + 2^-22 + 5 * 2^-24 =
    1.3e-6 of the sum of p v (no value is negative)."""
    hk, d, n = 512, 64, 64
    rng = np.random.default_rng(near + 200)
    ref = cache_tests.random_cache(rng, hk, n, d)
    ref.k[:], ref.v = 0, np.abs(ref.v)
    ref.vs[:] = np.ldexp(1 + rng.random(ref.vs.shape), near + rng.integers(0, 2, ref.vs.shape)).astype(np.float32)
    q = rng.standard_normal((T, hk, d)).astype(np.float32)
    got = cache_tests.run(gpu, rt, q, ref, np.full(T, n - 1), None, room)
    v = ref.values()[1]
    off = (np.abs(got - v.mean(1)) / v.mean(1)).max()
    assert off <= 1.3e-6, off


@pytest.mark.parametrize("T,room", [(1, None), (3, 1 << 18), (160, 1 << 18)])
@pytest.mark.parametrize("power", [-130, -126, -118, -100, 90])
def test_queries_and_key_scales_at_opposite_ends(gpu, rt, T, room, power):
    """Queries down to subnormal numbers over keys near float32's largest, and the
    other way round, whose scores are ordinary: within the bound of any others."""
    rng = np.random.default_rng(power + 200)
    ref = cache_tests.random_cache(rng, 2, 500, 64, spread=0.3)
    q = rng.standard_normal((T, 4, 64)).astype(np.float32)
    q, by = np.ldexp(q, power).astype(np.float32), -power if power > 0 else min(-power, 123)
    ref.ks[:] = np.ldexp(ref.ks, by)
    kend = 499 - np.arange(T)[::-1]
    got = cache_tests.run(gpu, rt, q, ref, kend, None, room)
    rows = sorted({0, T // 2, T - 1})
    want, bound = attention_bound.attention(q[rows], ref, kend[rows])
    off = np.abs(got[rows] - want)
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("T,n,room", [(1, 300, None), (1, 6000, None), (130, 600, 1 << 18)])
@pytest.mark.parametrize("power", [12, 20, 23, 26, 27, 28, 30, 40, 60, 100])
def test_scores_far_past_the_exponential(gpu, rt, T, n, room, power):
    """Scores up to 2^power (of log2 weights): a row is its best key's value, where
    float32 tells it from the next (40 and 2^-20 of its size apart). The best
    weight is 2^8 to 2^15 in two parts, of error 2^-22, the sum takes a reciprocal
    twice: 2^-20 of the value. The n others weigh at most 2^-40 of it each, with a
    scale in common: n 2^-40 of the largest value more."""
    rng = np.random.default_rng(power)
    ref = cache_tests.random_cache(rng, 1, n, 64)
    q = rng.standard_normal((T, 4, 64)).astype(np.float32)
    k, v = (x[0] for x in ref.values())
    scores = lambda q: q.astype(np.float64) @ k.T * np.log2(np.e) / 8  # noqa: E731
    q = (q * (2.0 ** power / np.abs(scores(q)).max())).astype(np.float32)
    z = scores(q)
    two = np.sort(z, -1)[..., -2:]
    clear = two[..., 1] - two[..., 0] > 40 + 2.0 ** -20 * two[..., 1]
    assert clear.any()
    got, want = cache_tests.run(gpu, rt, q, ref, np.full(T, n - 1), None, room)[clear], v[z.argmax(-1)][clear]
    assert (np.abs(got - want) <= 2.0 ** -20 * np.abs(want) + n * 2.0 ** -40 * np.abs(v).max()).all()
