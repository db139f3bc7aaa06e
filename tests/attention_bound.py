"""Attention over an 8-bit cache in 64 bits, with a bound for each output that
an evaluation "to float32 accuracy" (include/mimg.h) keeps and that a lost low
part, block or key does not.

out = sum_j p_j v_j / L, p_j = 2^(z_j - max z), z_j = q.k_j log2(e) / sqrt(d), L
= sum p. An error dz_j of an exponent moves out by p_j (v_j - out) ln 2 dz_j /
L, to first order; all terms below are of this form or relative to a sum.
Roundings are taken as independent where they are (of different numbers), so
they add as squares; LAMBDA times the root of the sum of the squared largest
roundings is more than ten deviations (a rounding of at most e has a deviation
of e / sqrt 3). With u = 2^-24:

 - q in two float16 parts, to 2^-22 of each element or 2^-39 of the row's
   largest: the same error for all keys, so it is added over them plainly
   (over the elements of the row as squares);
 - the scores' factor and the block's (two products, a constant): 4 u |z_j|,
   plainly;
 - the score's sum, at most dp roundings (d padded to 64s) of at most the
   largest partial sum;
 - the exponent: fused multiply-add and the block's offset, u times a magnitude
   of at most |z_j - max z| + 32; the exponential, one unit in the last place; the
   weight in two parts, 2^-22. Those of a block's keys may be the same, so they
   are added plainly in a block and as squares over blocks;
 - weights below 2^-22 of the largest end at 2^-44 of it, counted with the
   value scales in both (w_j = p_j * scale of its block): times the value's
   integer;
 - the sums over the keys: 8 roundings a block of at most the largest partial
   sum, counted with four times the root of the summed squares (partial sums
   of some of the keys); the sum of weights; 32 u for moves of the maximum,
   joins and the division."""
import numpy as np

U = 2.0 ** -24
LAMBDA = 6


def seen(kend, kstart, max_keys, context, t):
    lo = 0 if kstart is None else min(max(int(kstart[t]), 0), context - 1)
    return lo, max(min(int(kend[t]) + 1 - lo, context - lo, max_keys or context), 0)


def attention(q, ref, kend, kstart=None, max_keys=None):
    """float64 out [T, H, d] of float32 q over a q8_ref.Cache without marks in
    what is seen, and the bound of each output."""
    T, H, d = q.shape
    G, dp = H // ref.k.shape[0], (d + 63) // 64 * 64
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for t in range(T):
        lo, n = seen(kend, kstart, max_keys, ref.context, t)
        if n == 0:
            continue
        at = slice(lo, lo + n)
        block = np.arange(lo, lo + n) // 32
        first = np.flatnonzero(np.diff(block, prepend=-1))
        for h in range(H):
            x = q[t, h].astype(np.float64)
            k = ref.k[h // G, at].astype(np.float64) * ref.ks[h // G].astype(np.float64)[block, None]
            ints, vs = ref.v[h // G, at].astype(np.float64), ref.vs[h // G].astype(np.float64)[block]
            v = ints * vs[:, None]
            c = np.log2(np.e) / np.sqrt(d)
            kx = k * x * c
            z = kx.sum(1)
            p = np.exp2(z - z.max())
            L = p.sum()
            pv = p[:, None] * v
            o = out[t, h] = pv.sum(0) / L
            dv = p[:, None] * np.abs(v - o)
            steady = np.log(2) * (LAMBDA * 2.0 ** -22 * np.sqrt((kx ** 2).sum(1)) +
                                  2.0 ** -39 * np.abs(x).max() * np.abs(k).sum(1) * c + 4 * U * np.abs(z))
            each = 2.0 ** -22 + 2 * U + np.log(2) * U * (np.abs(z - z.max()) + 32 + np.sqrt(dp) * np.abs(np.cumsum(kx, 1)).max(1))
            blocks = np.add.reduceat(dv * each[:, None], first, 0)
            w = p * vs
            least = 2.0 ** -44 * w.max() * np.sqrt((ints ** 2).sum(0))
            part = np.abs(np.cumsum(pv, 0)).max(0) / L + 4 * np.sqrt((pv ** 2).sum(0)) / L
            nb = len(first)
            bound[t, h] = ((dv * steady[:, None]).sum(0) + LAMBDA * (np.sqrt((blocks ** 2).sum(0)) + least)) / L + \
                LAMBDA * U * (np.sqrt(8 * nb + 64) * part + np.sqrt(nb + 64) * np.abs(o)) + 32 * U * np.abs(o) + 1e-37
    return out, bound


def sink_cache(rng, cache, q, gap):
    """Ordinary integers and scales in the q8_ref.Cache, values with a mean of half
    their deviation, but a first key that q [T, H, d] (float32, turned towards it
    here) scores `gap` nats above the rest, its value zero: what a trained
    model's first token does. Returns the new q."""
    T, H, d = q.shape
    for name, mean in (("k", 0), ("v", 18)):
        ints = np.clip(np.rint(rng.standard_normal(getattr(cache, name).shape) * 36 + mean), -127, 127)
        setattr(cache, name, ints.astype(np.int8))
        scales = np.exp(rng.standard_normal(getattr(cache, name + "s").shape) * 0.3) / 36
        setattr(cache, name + "s", scales.astype(np.float32))
    hk = cache.k.shape[0]
    to = np.sign(rng.standard_normal((hk, d)))
    cache.ks[:, 0], cache.vs[:, 0] = 1 / 36, 1 / 36
    cache.k[:, 0], cache.v[:, 0] = (to * 120).astype(np.int8), 0
    rest = np.sqrt(2 * np.log(cache.context + 2))  # about the largest of the others' scores, whose deviation is near 1
    lean = (gap + rest) / (120 / 36 * np.sqrt(d))
    return (q + np.repeat(to, H // hk, 0) * lean).astype(np.float32)
