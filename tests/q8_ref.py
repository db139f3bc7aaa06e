"""Plain 64-bit restatements of the 8-bit cache's operators and of the log
probabilities, from their definitions in include/mimg.h (numpy)."""
import numpy as np

FLOOR = 2.0 ** -96


class Cache:
    """Integers, float32 scales and marks of [kv_heads, context, d]."""

    def __init__(self, kv_heads, context, d):
        nb = (context + 31) // 32
        self.context = context
        self.k, self.v = (np.zeros((kv_heads, nb * 32, d), np.int8) for _ in range(2))
        self.ks, self.vs = (np.zeros((kv_heads, nb), np.float32) for _ in range(2))
        self.bad = np.zeros((kv_heads, nb), np.uint32)

    def store(self, k, v, index):
        """k, v float32 [T, kv_heads, d]."""
        last = {int(i): t for t, i in enumerate(index) if 0 <= i < self.context}  # of one index the later row
        for b in sorted({i // 32 for i in last}):
            rows = {i % 32: t for i, t in last.items() if i // 32 == b}
            for h in range(self.k.shape[0]):
                bad = 0 if 0 in rows else int(self.bad[h, b])
                for e, t in rows.items():
                    ok = np.isfinite(k[t, h]).all() and np.isfinite(v[t, h]).all()
                    bad = bad & ~(1 << e) | (0 if ok else 1 << e)
                self.bad[h, b] = bad
                for q, s, x in ((self.k, self.ks, k), (self.v, self.vs, v)):
                    new = {e: np.where(np.isfinite(x[t, h]), x[t, h], 0).astype(np.float64) for e, t in rows.items()}
                    amax = max(np.abs(r).max() for r in new.values())
                    was = 0.0 if 0 in rows else float(s[h, b])
                    scale = max(was, max(float(np.float32(amax / 127)), FLOOR) if amax > 0 else 0.0)
                    at = slice(32 * b, 32 * b + 32)
                    kept = q[h, at].astype(np.float64) * was
                    if 0 in rows:
                        kept[:] = 0
                    for e, r in new.items():
                        kept[e] = r
                    q[h, at] = np.clip(np.rint(kept / scale), -127, 127) if scale > 0 else 0
                    s[h, b] = scale

    def values(self):
        """(k, v) float64 [kv_heads, context, d]; marked entries NaN."""
        out = []
        for q, s in ((self.k, self.ks), (self.v, self.vs)):
            x = q.astype(np.float64) * np.repeat(s.astype(np.float64), 32, 1)[..., None]
            marks = (self.bad[..., None] >> np.arange(32, dtype=np.uint32)) & 1
            x[marks.reshape(x.shape[0], -1).astype(bool)] = np.nan
            out.append(x[:, :self.context])
        return out


def attention(q, k, v, kend, kstart=None, max_keys=None):
    """float64 [T, H, d] over k, v [kv_heads, context, d], and the bound of a
    float32 evaluation for each (t, h): scores as sums of d products of 22-bit
    parts, weights by a float32 exponential, sums over the keys."""
    T, H, d = q.shape
    G, C = H // k.shape[0], k.shape[1]
    out, bound = np.zeros(q.shape), np.zeros((T, H))
    for t in range(T):
        lo = 0 if kstart is None else min(max(int(kstart[t]), 0), C - 1)
        n = min(int(kend[t]) + 1 - lo, C - lo, max_keys or C)
        if n <= 0:
            continue
        for h in range(H):
            kk, vv = k[h // G, lo:lo + n], v[h // G, lo:lo + n]
            x = q[t, h].astype(np.float64)
            s = kk @ x / np.sqrt(d)
            with np.errstate(invalid="ignore"):
                p = np.exp(s - s.max())
                out[t, h] = p @ vv / p.sum()
                # products to 2^-22, a sum of d terms, the scale; twice (weights and
                # their sum); the exponent's own rounding (|log2 of a weight| below
                # 2^7: 2^-17 at most where it counts), the sums over n keys
                a = (np.abs(kk) @ np.abs(x) / np.sqrt(d)).max()
                eps = 2 * a * (2.0 ** -22 + (d + 4) * 2.0 ** -24) + (n + 128) * 2.0 ** -24
                bound[t, h] = eps * np.abs(vv).max()
    return out, bound


def logprobs(x, targets, top):
    """(logprob, entropy, top_ids, top_logprobs), float64, of finite or -inf rows."""
    x = x.astype(np.float64)
    m = x.max(-1, keepdims=True)
    e = np.exp(x - m)
    lp = x - m - np.log(e.sum(-1, keepdims=True))
    p = np.exp(lp)
    ent = -np.where(p > 0, p * np.where(p > 0, lp, 0), 0).sum(-1)
    n = x.shape[1]
    given = np.array([lp[r, t] if 0 <= t < n else 0.0 for r, t in enumerate(targets)])
    ids = np.argsort(-x, axis=-1, kind="stable")[:, :top]
    return given, ent, ids, np.take_along_axis(lp, ids, -1)
