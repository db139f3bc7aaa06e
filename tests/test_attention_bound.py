"""attention_bound.py's bound can fail: evaluations that lose a low part, a block
of keys or one key, or see one too many, pass it in no case here; one with all
parts (24 bits of score and 22 of weight, else exact) stays far below."""
import numpy as np
import pytest

import attention_bound
import q8_ref


def random_cache(rng, hk, context, d):
    ref = q8_ref.Cache(hk, context, d)
    for name in ("k", "v"):
        ints = np.clip(np.rint(rng.standard_normal(ref.k.shape) * 36), -127, 127)
        setattr(ref, name, ints.astype(np.int8))
        setattr(ref, name + "s", (np.exp(rng.standard_normal(ref.ks.shape) * 0.5) / 36).astype(np.float32))
    return ref


def f16(x):
    return x.astype(np.float16).astype(np.float64)


def f16_towards_zero(x):
    h = x.astype(np.float16)
    return np.where(np.abs(h.astype(np.float64)) > np.abs(x), np.nextafter(h, np.float16(0)), h).astype(np.float64)


def one_scale(y):
    """Two parts that both end at 2^-24, towards zero."""
    h = f16_towards_zero(y)
    return h + f16_towards_zero(y - h)


WEIGHTS = dict(two=lambda y: f16(y) + f16((y - f16(y)) * 2048) / 2048, one=f16, one_towards_zero=f16_towards_zero, one_scale=one_scale)


def evaluate(q, ref, kend, q_parts=2, weights="two", drop=None, more=0):
    """Attention with q and the weights in float16 parts, else in 64 bits;
    without block `drop`, with `more` keys at the end."""
    T, H, d = q.shape
    out = np.zeros(q.shape)
    for t in range(T):
        n = int(kend[t]) + 1 + more
        block = np.arange(n) // 32
        for h in range(H):
            hk = h // (H // ref.k.shape[0])
            x = q[t, h].astype(np.float64)
            e = 15 - np.frexp(np.abs(x).max())[1]
            x = np.ldexp(x, e)
            x = np.ldexp(f16(x) + (f16(x - f16(x)) if q_parts == 2 else 0), -e)
            k = ref.k[hk, :n] * ref.ks[hk].astype(np.float64)[block, None]
            vs = ref.vs[hk].astype(np.float64)[block]
            w = k @ x * np.log2(np.e) / np.sqrt(d) + np.log2(vs)
            y = np.exp2(w - w.max() + 8)
            if drop is not None:
                y[block == drop % (block[-1] + 1)] = 0
            out[t, h] = WEIGHTS[weights](y) @ ref.v[hk, :n] / (y / vs).sum()
    return out


@pytest.mark.parametrize("H,hk,d,n", [(4, 1, 64, 250), (4, 2, 64, 1400), (4, 2, 128, 900), (3, 1, 64, 1500), (4, 4, 192, 700),
                                      (4, 2, 256, 4000), (3, 3, 80, 1300), (4, 2, 128, 2500), (4, 2, 128, 6000),
                                      (3, 1, 64, 20001), (4, 1, 64, 181), (4, 2, 80, 77), (4, 1, 256, 700)])
def test_what_the_bound_tells_apart(H, hk, d, n):
    rng = np.random.default_rng(n)
    ref = random_cache(rng, hk, n, d)
    q = rng.standard_normal((2, H, d)).astype(np.float32)
    kend = np.array([n - 3, n - 2])
    want, bound = attention_bound.attention(q, ref, kend)
    ratio = lambda **kw: (np.abs(evaluate(q, ref, kend, **kw) - want) / bound).max()  # noqa: E731
    assert ratio() < 0.1
    wrong = [dict(weights="one"), dict(weights="one_towards_zero"), dict(q_parts=1), dict(weights="one", q_parts=1), dict(drop=0),
             dict(drop=-1), dict(drop=n // 64), dict(more=1), dict(more=-1)]
    for kw in wrong:
        assert ratio(**kw) > 1, kw


@pytest.mark.parametrize("H,hk,d,n", [(2, 1, 64, 20000), (4, 2, 128, 2000), (2, 2, 80, 40), (2, 1, 256, 2500)])
@pytest.mark.parametrize("gap", [10, 14, 18])
def test_behind_a_key_that_outweighs_the_rest(H, hk, d, n, gap):
    rng = np.random.default_rng(n + gap)
    ref = q8_ref.Cache(hk, n, d)
    q = attention_bound.sink_cache(rng, ref, rng.standard_normal((2, H, d)).astype(np.float32), gap)
    kend = np.array([n - 3, n - 2])
    want, bound = attention_bound.attention(q, ref, kend)
    ratio = lambda **kw: (np.abs(evaluate(q, ref, kend, **kw) - want) / bound).max()  # noqa: E731
    assert ratio() < 0.5  # (weights that end at 2^-44 of the largest among them)
    assert ratio(weights="one_scale") > 5 and ratio(q_parts=1) > 1


def test_a_row_that_sees_nothing_and_windows():
    """Zeros, and the keys from kstart on up to max_keys: those of a cache cut
    out at whole blocks."""
    rng = np.random.default_rng(3)
    ref = random_cache(rng, 1, 320, 64)
    q = rng.standard_normal((3, 2, 64)).astype(np.float32)
    got, bound = attention_bound.attention(q, ref, np.array([70, 300, 9]), np.array([71, 64, 0]), 100)
    assert not got[0].any() and not bound[0].any() and (bound[1:] > 0).all()
    cut = q8_ref.Cache(1, 256, 64)
    cut.k, cut.v, cut.ks, cut.vs = ref.k[:, 64:], ref.v[:, 64:], ref.ks[:, 2:], ref.vs[:, 2:]
    want, same = attention_bound.attention(q[1:2], cut, np.array([99]))
    assert np.array_equal(got[1], want[0]) and np.array_equal(bound[1], same[0])
    plain, _ = q8_ref.attention(q, *ref.values(), np.array([70, 300, 9]), np.array([71, 64, 0]), 100)
    assert np.allclose(got, plain, rtol=1e-9, atol=1e-12)
