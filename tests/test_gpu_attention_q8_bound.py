"""Attention over the 8-bit cache within attention_bound's bound, which a lost low
part, block or key does not keep (test_attention_bound.py): each kernel, its
splits and joins, on ordinary inputs."""
import numpy as np
import pytest

import attention_bound
import q8_ref
import test_gpu_cache_q8 as cache_tests

pytestmark = pytest.mark.gpu
rt = cache_tests.rt


def check(got, ref, q, kend, kstart, room, rows, heads):
    """Some rows and heads, each with its kv head's cache."""
    H, hk = q.shape[1], ref.k.shape[0]
    for h in heads:
        at = slice(h // (H // hk), h // (H // hk) + 1)
        one = q8_ref.Cache(1, ref.context, q.shape[2])
        one.k, one.v, one.ks, one.vs = ref.k[at], ref.v[at], ref.ks[at], ref.vs[at]
        want, bound = attention_bound.attention(q[rows, h:h + 1], one, kend[rows], None if kstart is None else kstart[rows], room)
        off = np.abs(got[rows, h:h + 1] - want)
        assert (off <= bound).all(), (h, (off / np.maximum(bound, 1e-37)).max())


# `room`: max_keys; far more than the cache holds means many splits, and from 64
# tokens the prompt kernel beside the other
@pytest.mark.parametrize("room", [None, 1 << 18])
@pytest.mark.parametrize("T,H,hk,d,slots,stride", [
    (1, 4, 1, 8, 1, 1), (1, 1, 1, 64, 1, 32), (1, 32, 8, 64, 1, 181), (1, 8, 2, 128, 1, 6000), (1, 3, 1, 64, 1, 20001),
    (1, 34, 2, 256, 1, 700), (2, 16, 2, 256, 1, 4000), (3, 14, 2, 64, 3, 500), (5, 40, 2, 80, 5, 77), (7, 3, 1, 64, 1, 1500),
    (8, 32, 8, 128, 8, 300), (20, 8, 2, 128, 1, 900), (33, 4, 4, 192, 1, 700), (63, 6, 6, 80, 1, 1300), (64, 4, 2, 64, 16, 70),
    (64, 8, 2, 128, 1, 2500), (65, 12, 4, 256, 2, 100), (100, 144, 1, 64, 1, 250), (109, 14, 2, 128, 3, 260),
    (128, 14, 2, 64, 1, 1400), (150, 16, 2, 128, 150, 13), (181, 14, 2, 64, 1, 181), (300, 6, 2, 192, 2, 400),
    (512, 32, 8, 128, 1, 2600), (700, 8, 1, 64, 1, 9000)])
def test_attention(gpu, rt, T, H, hk, d, slots, stride, room):
    rng = np.random.default_rng(T * 37 + H + stride)
    C = slots * stride
    ref = cache_tests.random_cache(rng, hk, C, d, spread=0.5)
    q = rng.standard_normal((T, H, d)).astype(np.float32)
    slot = np.sort(np.arange(T) % slots)
    start = slot * stride
    if slots == 1:
        end = np.maximum(C - T, 0) + np.arange(T)
    else:
        end = start + rng.integers(0, stride, T)
        end[-1] = start[-1] + stride - 1
    kstart = start if slots > 1 else None
    got = cache_tests.run(gpu, rt, q, ref, end, kstart, room)
    rows = sorted({0, T // 3, T // 2, T - 2 if T > 1 else 0, T - 1})
    check(got, ref, q, end, kstart, room, rows, sorted({0, H // 2, H - 1}))


def test_one_row_over_a_long_cache(gpu, rt):
    """64 splits of 60 blocks and more, four waves each."""
    rng = np.random.default_rng(9)
    ref = cache_tests.random_cache(rng, 1, 131072, 64, spread=0.3)
    q = rng.standard_normal((1, 4, 64)).astype(np.float32)
    end = np.array([131000])
    check(cache_tests.run(gpu, rt, q, ref, end), ref, q, end, None, None, [0], [0, 3])
