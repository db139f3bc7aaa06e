"""Attention over the 8-bit cache where one key outweighs the rest by 10 to 18
nats and has a value of zero, so that the outputs are those of weights down to
2^-30 of the largest: within attention_bound's bound, which is relative to the
sum of p |v| there."""
import numpy as np
import pytest

import attention_bound
import q8_ref
import test_gpu_cache_q8 as cache_tests

pytestmark = pytest.mark.gpu
rt = cache_tests.rt


# (prompts that the keys of one workgroup reach to the end, prompts and rows in
# splits, rows packed together, single rows; each padded head size)
@pytest.mark.parametrize("T,H,hk,d,n,room", [
    (2048, 32, 1, 64, 100000, None), (2048, 32, 1, 128, 8192, None), (512, 8, 2, 128, 2000, None), (130, 4, 1, 256, 2500, 1 << 18),
    (96, 6, 2, 192, 3000, 1 << 18), (64, 4, 1, 64, 100000, None), (20, 8, 2, 128, 900, 1 << 18), (1, 4, 1, 64, 100000, None),
    (1, 8, 2, 128, 2000, None), (3, 2, 2, 80, 40, None)])
@pytest.mark.parametrize("gap", [10, 14, 18])
def test_behind_a_key_that_outweighs_the_rest(gpu, rt, T, H, hk, d, n, room, gap):
    rng = np.random.default_rng(T + n + gap)
    ref = q8_ref.Cache(hk, n, d)
    q = attention_bound.sink_cache(rng, ref, rng.standard_normal((T, H, d)).astype(np.float32), gap)
    kend = n - T + np.arange(T) if T <= n else np.arange(T) % n
    got = cache_tests.run(gpu, rt, q, ref, kend, None, room)
    # of a long call some rows and heads of every kv head
    rows = sorted({0, T // 2, T - 1})
    heads = sorted({0, H // 2, H - 1}) if n < 50000 else [H - 1]
    for h in heads:
        one = q8_ref.Cache(1, n, d)
        hh = h // (H // hk)
        one.k, one.v, one.ks, one.vs = ref.k[hh:hh + 1], ref.v[hh:hh + 1], ref.ks[hh:hh + 1], ref.vs[hh:hh + 1]
        want, bound = attention_bound.attention(q[rows, h:h + 1], one, kend[rows])
        off = np.abs(got[rows, h:h + 1] - want)
        assert (off <= bound).all(), (h, (off / bound).max())
