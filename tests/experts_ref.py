"""The operators of a mixture of experts restated in float64 from their
definitions (include/mimg.h): the router, the plan, the experts' products with
the bound of their float32 chains, swiglu of two of them, the weighted sum."""
import numpy as np

import mimref

EPS = 2.0 ** -24
BLOCK = {mimref.Q4_K: 256, mimref.Q6_K: 256, mimref.Q8_0: 32}


def plan(ids, experts):
    """(first [experts + 1], order, expert) of choices ids [T, top]."""
    flat = np.asarray(ids).reshape(-1).astype(np.int64)
    flat = np.where((flat < 0) | (flat >= experts), experts, flat)
    first = np.array([(flat < e).sum() for e in range(experts + 1)], np.int32)
    return first, np.argsort(flat, kind="stable").astype(np.int32), np.where(flat == experts, -1, flat).astype(np.int32)


def packed_plan(ids, experts):
    """The plan as the library lays it out."""
    first, order, expert = plan(ids, experts)
    up = lambda n: (n + 63) // 64 * 64  # noqa: E731
    out = np.zeros(up(experts + 1) + up(order.size) + order.size, np.int32)
    out[:experts + 1] = first
    out[up(experts + 1):up(experts + 1) + order.size] = order
    out[up(experts + 1) + up(order.size):] = expert
    return out


def route(x, router, top, normalize):
    """(ids, weights in float64): NaN behind all, equal logits by the index."""
    with np.errstate(all="ignore"):
        logits = x.astype(np.float64) @ router.astype(np.float64).T
        key = np.where(np.isnan(logits), np.inf, -logits)
        # lexsort: NaN last of all, then falling, then the index
        ids = np.stack([np.lexsort((np.arange(r.size), k, np.isnan(r))) for r, k in zip(logits, key)])[:, :top]
        value = np.take_along_axis(logits, ids, 1)
        e = np.exp((value if normalize else logits) - value[:, :1])
        return ids.astype(np.int32), np.exp(value - value[:, :1]) / e.sum(-1, keepdims=True)


def parts(dt, raw, n, k):
    """Weight rows as (integers [n, blocks, block], scale [n, blocks], mins and
    their scale likewise or None): a weight is integer * scale - min * its."""
    raw = np.asarray(raw, np.uint8)
    if dt == mimref.Q8_0:
        b = raw.reshape(n, k // 32, 34)
        return b[..., 2:].view(np.int8).astype(np.float64), b[..., :2].copy().view(np.float16)[..., 0].astype(np.float64), None, None
    if dt == mimref.Q6_K:
        b = raw.reshape(n, k // 256, 210)
        ql, qh = b[..., :128].reshape(n, -1, 2, 2, 32).astype(int), b[..., 128:192].reshape(n, -1, 2, 1, 32).astype(int)
        q = np.concatenate([ql & 15, ql >> 4], 3) | ((qh >> np.array([0, 2, 4, 6]).reshape(4, 1)) & 3) << 4
        sc = b[..., 192:208].view(np.int8).astype(np.float64)
        return ((q - 32).reshape(n, -1, 16, 16) * sc[..., None]).reshape(n, -1, 256), \
            b[..., 208:].copy().view(np.float16)[..., 0].astype(np.float64), None, None
    b = raw.reshape(n, k // 256, 144)
    d = b[..., :4].copy().view(np.float16).astype(np.float64)
    h = b[..., 4:16].astype(int)
    sc = np.concatenate([h[..., :4] & 63, h[..., 8:] & 15 | h[..., :4] >> 6 << 4], -1)
    m = np.concatenate([h[..., 4:8] & 63, h[..., 8:] >> 4 | h[..., 4:8] >> 6 << 4], -1)
    q = b[..., 16:].reshape(n, -1, 4, 1, 32).astype(int)
    q = np.concatenate([q & 15, q >> 4], 3).reshape(n, -1, 8, 32)
    return (q * sc[..., None]).reshape(n, -1, 256).astype(np.float64), d[..., 0], np.repeat(m, 32, -1).astype(np.float64), d[..., 1]


def acts(x, block):
    """(integers [rows, blocks, block], scales [rows, blocks]) of rows in 8 bits."""
    b = x.astype(np.float64).reshape(x.shape[0], -1, block)
    amax = np.abs(b).max(-1)
    q = np.rint(127 * b / np.where(amax > 0, amax, 1)[..., None])
    return q, (amax.astype(np.float32) / np.float32(127)).astype(np.float64)


def product(x, raw, dt, n, k):
    """(x . W^T in float64 on the 8-bit rows, the bound of the float32 chain).
    A block's term S d dx has S and d dx rounded (2 EPS of it), a step of the
    chain EPS of what it has so far, and Q4_K's two chains are subtracted: at
    most (blocks + 3) EPS of the terms' sizes, taken 1.01 times for products of
    roundings."""
    q, dx = acts(x, BLOCK[dt])
    w, d, m, dm = parts(dt, raw, n, k)
    term = np.einsum("rbk,nbk->rnb", q, w) * d[None] * dx[:, None]
    total, size = term.sum(-1), np.abs(term).sum(-1)
    if m is not None:
        term = np.einsum("rbk,nbk->rnb", q, m) * dm[None] * dx[:, None]
        total, size = total - term.sum(-1), size + np.abs(term).sum(-1)
    return total, 1.01 * (d.shape[1] + 3) * EPS * size


def swiglu(g, ge, u, ue):
    """silu(g) * u and a bound for g and u that are ge and ue off: |silu'| is
    at most 1.1, and the function's own float32 steps 12 EPS (an exponential of
    a few, two products, two additions, a division, the last product)."""
    s = g / (1 + np.exp(-g))
    return s * u, 1.1 * ge * (np.abs(u) + ue) + np.abs(s) * ue + 12 * EPS * (np.abs(s) + 1.1 * ge) * (np.abs(u) + ue)
