"""Few pairs of Q8_0 experts where a token has more than two of them: each by
itself (experts_q8.hip), against float64 and bit for bit against the tiles, which
take the same tokens 64 times over."""
import numpy as np
import pytest

import experts_ref as ref
from test_gpu_experts import Layer, Q8_0, acts_for, bits, check_combine, check_swiglu, choices, rt, run_combine, run_swiglu  # noqa: F401

pytestmark = pytest.mark.gpu
MANY = 64

# experts, n, k, T, top, choices: 8 to 32 sets of a workgroup, some without an
# expert, one expert twice; 5 to 64 pairs
SUMS = [(64, 20, 96, 2, 8, "even"), (64, 33, 800, 3, 5, "even"), (128, 33, 800, 5, 8, "padded"), (128, 12, 544, 8, 8, "again"),
        (64, 9, 512, 1, 32, "even"), (64, 9, 1408, 1, 12, "padded"), (48, 7, 1056, 2, 9, "even"), (160, 6, 32, 64, 1, "padded")]
# ... and one to sixteen pairs of several tokens, rows that are no multiple of four
SWIGLUS = [(64, 20, 96, 2, 8, "even"), (40, 33, 800, 3, 4, "padded"), (32, 35, 1408, 4, 4, "again"), (16, 21, 288, 8, 1, "even"),
           (12, 9, 64, 3, 2, "padded"), (64, 130, 512, 1, 16, "even")]


def many(a):
    return np.tile(a, (MANY, 1))


@pytest.mark.parametrize("experts,n,k,T,top,what", SUMS)
def test_sum(gpu, rt, oracle, experts, n, k, T, top, what):  # noqa: F811
    assert T * top <= 4 or T * top <= 32 and 2 * experts >= 3 * T * top or T * top <= 64 and experts >= 2 * T * top
    down = Layer(gpu, oracle, Q8_0, experts, n, k, 1)
    h, ids = acts_for(2, T * top, k), choices(3, T, top, experts, what)
    assert (ids >= 0).any()
    weights = np.random.default_rng(4).random((T, top), np.float32)
    got = run_combine(gpu, rt, down, h, weights, ids)
    check_combine(got, oracle, down, h, weights, ids)
    np.testing.assert_array_equal(bits(many(got)), bits(run_combine(gpu, rt, down, many(h), many(weights), many(ids))))


@pytest.mark.parametrize("experts,n,k,T,top,what", SWIGLUS)
def test_swiglu(gpu, rt, oracle, experts, n, k, T, top, what):  # noqa: F811
    assert T * top <= 4 or T * top <= 16 and experts >= 2 * T * top
    gate, up = (Layer(gpu, oracle, Q8_0, experts, n, k, seed) for seed in (5, 6))
    x, ids = acts_for(7, T, k), choices(8, T, top, experts, what)
    assert (ids >= 0).any()
    got = run_swiglu(gpu, rt, gate, up, x, ids)
    check_swiglu(got, oracle, gate, up, x, ids)
    np.testing.assert_array_equal(bits(many(got)), bits(run_swiglu(gpu, rt, gate, up, many(x), many(ids))))


@pytest.mark.parametrize("top", [9, 20, 32])
def test_refused_rows_of_many_sets(gpu, rt, oracle, top):  # noqa: F811
    """Pairs whose row of h is beyond 2^60 are float32 products of the decoded
    weights, 32 chains of k / 32 steps and five additions: each step EPS of what
    it has so far, the weight's decoding and its product inside one EPS more."""
    k, n, experts = 512, 13, 64
    down = Layer(gpu, oracle, Q8_0, experts, n, k, 9)
    h, ids = acts_for(10, 2 * top, k), choices(11, 2, top, experts)
    if top == 32:
        h, ids = h[:top], ids[:1]
    T = len(ids)
    weights = np.random.default_rng(12).random((T, top), np.float32)
    refused = [0, 8, top - 1]  # (rows of the sets from 8 on are a workgroup's second turn)
    h[refused, 5] = 2.0 ** 61
    got = run_combine(gpu, rt, down, h, weights, ids)
    np.testing.assert_array_equal(bits(many(got)), bits(run_combine(gpu, rt, down, many(h), many(weights), many(ids))))
    total, bound = np.zeros((T, n)), np.zeros((T, n))
    for t in range(T):
        size = np.zeros(n)
        for j in range(top):
            p, e = t * top + j, ids[t, j]
            if p in refused:
                term = oracle.dequantize(Q8_0, down.raw[e], n * k).reshape(n, k).astype(np.float64) * h[p].astype(np.float64)
                y, b = term.sum(-1), 1.01 * (k // 32 + 7) * ref.EPS * np.abs(term).sum(-1)
            else:
                y, b = (v[0] for v in ref.product(h[p:p + 1], down.raw[e], Q8_0, n, k))
            w = np.float64(weights[t, j])
            total[t] += w * y
            bound[t] += w * b
            size += w * (np.abs(y) + b)
        bound[t] = bound[t] * (1 + 2 * top * ref.EPS) + 1.01 * top * ref.EPS * size
    assert (np.abs(got - total) <= bound).all()
