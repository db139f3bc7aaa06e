"""Stores into the 8-bit cache and reads from it (cache_q8.hip), and attention
over it (attention_q8.hip), against the 64-bit restatements of q8_ref.py: the
cache's integers, scales and marks exactly, attention within the bound of a
float32 evaluation that q8_ref.attention derives."""
import numpy as np
import pytest

import q8_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt(gpu):
    import hiprt

    return hiprt


def dev(rt, a):
    return rt.DeviceBuffer.from_array(np.ascontiguousarray(a))


class DeviceCache:
    def __init__(self, gpu, rt, hk, context, d):
        self.gpu, self.rt, self.hk, self.context, self.d = gpu, rt, hk, context, d
        self.buf = rt.DeviceBuffer(gpu.cache_q8_bytes(hk, context, d) + 64)
        self.buf.zero()
        self.s = rt.Stream()

    def store(self, k, v, index):
        bufs = [dev(self.rt, a) for a in (k, v, np.asarray(index, np.int64))]
        self.gpu.kv_store_q8_dev(*(b.ptr for b in bufs), len(index), self.hk, self.d, self.context, self.buf.ptr, self.s.handle)
        self.s.sync()

    def raw(self):
        return self.buf.download(np.uint8)

    def parts(self):
        return self.gpu.unpack_cache_q8(self.raw()[:-64], self.hk, self.context, self.d)

    def load(self, index):
        T = len(index)
        k, v = (self.rt.DeviceBuffer(T * self.hk * self.d * 4) for _ in range(2))
        i = dev(self.rt, np.asarray(index, np.int64))
        self.gpu.kv_load_q8_dev(self.buf.ptr, i.ptr, T, self.hk, self.d, self.context, k.ptr, v.ptr, self.s.handle)
        self.s.sync()
        return tuple(b.download(np.float32).reshape(T, self.hk, self.d) for b in (k, v))


def check_cache(dc, ref):
    k, ks, v, vs, bad = dc.parts()
    live_k, live_v = np.repeat(ref.ks > 0, 32, 1)[:, :ref.context], np.repeat(ref.vs > 0, 32, 1)[:, :ref.context]
    assert np.array_equal(ks, ref.ks) and np.array_equal(vs, ref.vs) and np.array_equal(bad, ref.bad)
    for got, want, live in ((k, ref.k, live_k), (v, ref.v, live_v)):  # (a scale of zero: any integers)
        assert np.array_equal(got[live], want[:, :ref.context][live]), np.argwhere((got != want[:, :ref.context]) & live[..., None])[:5]
    assert not dc.raw()[-64:].any()  # nothing past the end


def values(rng, T, hk, d):
    x = rng.standard_normal((T, hk, d)).astype(np.float32)
    return x * np.exp(rng.standard_normal((T, hk, 1))).astype(np.float32)


@pytest.mark.parametrize("hk,d,C", [(2, 64, 128), (1, 128, 100), (3, 8, 70), (2, 80, 64), (1, 192, 96), (2, 256, 130), (8, 128, 300)])
def test_appends(gpu, rt, hk, d, C):
    """A prompt, tokens one by one over block borders, a jump back into the
    middle, a new sequence from the first entry on, the last partial block."""
    rng = np.random.default_rng(C * 7 + d)
    dc, ref = DeviceCache(gpu, rt, hk, C, d), q8_ref.Cache(hk, C, d)
    steps = [range(0, min(45, C)), *([i] for i in range(45, 50) if i < C), [20, 21], range(0, 3), range(C - 7, C), [C - 2]]
    for index in steps:
        index = list(index)
        k, v = values(rng, len(index), hk, d), values(rng, len(index), hk, d)
        dc.store(k, v, index)
        ref.store(k, v, index)
        check_cache(dc, ref)
    got = dc.load(list(range(C)) + [-1, C, 5])
    want = [np.float32(x).transpose(1, 0, 2) for x in ref.values()]
    for g, w in zip(got, want):
        assert np.array_equal(g[:C], w.astype(np.float32)) and not g[C:C + 2].any() and np.array_equal(g[C + 2], w[5])


@pytest.mark.parametrize("T", [1, 2, 31, 33, 200, 700, 1500, 2600])
def test_indices_in_any_order(gpu, rt, T):
    """Shuffled rows, the same index twice and more, rows outside the cache
    (its last, partial block's unused entries too), many rows a block."""
    hk, d, C = 2, 64, 333
    rng = np.random.default_rng(T)
    dc, ref = DeviceCache(gpu, rt, hk, C, d), q8_ref.Cache(hk, C, d)
    for _ in range(3):
        index = rng.integers(-3, C + 19, T)
        k, v = values(rng, T, hk, d), values(rng, T, hk, d)
        dc.store(k, v, index)
        ref.store(k, v, index)
        check_cache(dc, ref)


def test_scales_and_marks(gpu, rt):
    """Zero rows, scales at the floor and near float32's largest, ties, values
    that are not finite, and marks that a later store clears."""
    hk, d, C = 2, 64, 96
    dc, ref = DeviceCache(gpu, rt, hk, C, d), q8_ref.Cache(hk, C, d)
    x = np.zeros((1, hk, d), np.float32)
    tie = x.copy()
    tie[0, :, 0], tie[0, :, 1:] = 127.0, np.arange(63, dtype=np.float32) / 2  # a scale of 1: halves
    bad = tie.copy()
    bad[0, 0, 7], bad[0, 1, 9] = np.nan, -np.inf
    one_head = tie.copy()
    one_head[0, 1, 3] = np.inf
    steps = [(x, x, [0]), (x, x, [1]), (x + 1e-38, x - 1e-30, [2]), (x + 3e38, x - 3.4e38, [3]), (tie, x, [32]), (bad, tie, [33]),
             (tie, one_head, [34]), (tie, tie, [33]), (x + 0.25, tie * 2, [35]), (bad, bad, [64]), (x + 1, x + 1, [65]), (x, x, [0])]
    for k, v, index in steps:
        dc.store(k, v, index)
        ref.store(k, v, index)
        check_cache(dc, ref)
    got = dc.load([33, 34, 64, 65])
    assert not np.isnan(got[0][0]).any() and np.isnan(got[0][1, 1]).all() and not np.isnan(got[0][1, 0]).any()
    assert np.isnan(got[1][2]).all() and not np.isnan(got[1][3]).any()


@pytest.mark.parametrize("H,hk,d,rotary,inter", [(4, 2, 64, 64, 1), (8, 8, 128, 128, 0), (6, 3, 80, 48, 0), (14, 2, 64, 32, 1),
                                                 (2, 1, 256, 256, 0), (1030, 1, 256, 64, 1), (600, 600, 8, 8, 0)])
@pytest.mark.parametrize("T", [1, 5, 70, 1100])
def test_rope_and_store_in_one_launch(gpu, rt, T, H, hk, d, rotary, inter):
    rng = np.random.default_rng(T + d)
    C = 128
    q, k, v = values(rng, T, H, d), values(rng, T, hk, d), values(rng, T, hk, d)
    pos = rng.integers(0, 5000, T).astype(np.int64)
    index = (np.arange(T) + 17).astype(np.int64)
    freq = dev(rt, 10000.0 ** (-2.0 * np.arange(rotary // 2) / rotary))
    one, two = DeviceCache(gpu, rt, hk, C, d), DeviceCache(gpu, rt, hk, C, d)
    dp, di, dv = dev(rt, pos), dev(rt, index), dev(rt, v)
    q1, k1, q2, k2 = dev(rt, q), dev(rt, k), dev(rt, q), dev(rt, k)
    gpu.rope_kv_q8_dev(q1.ptr, k1.ptr, dv.ptr, dp.ptr, di.ptr, freq.ptr, T, H, hk, d, rotary, inter, C, one.buf.ptr, one.s.handle)
    one.s.sync()
    gpu.rope_dev(q2.ptr, dp.ptr, freq.ptr, T, H, d, rotary, inter, two.s.handle)
    gpu.rope_dev(k2.ptr, dp.ptr, freq.ptr, T, hk, d, rotary, inter, two.s.handle)
    gpu.kv_store_q8_dev(k2.ptr, dv.ptr, di.ptr, T, hk, d, C, two.buf.ptr, two.s.handle)
    two.s.sync()
    assert np.array_equal(one.raw(), two.raw())
    assert np.array_equal(q1.download(np.uint32), q2.download(np.uint32))
    assert np.array_equal(k1.download(np.float32).reshape(k.shape), k)  # k as it was


# ---- attention ---------------------------------------------------------------

def random_cache(rng, hk, context, d, spread=0.0):
    """int8 values and scales; spread: of the scales between blocks, in powers
    of e."""
    ref = q8_ref.Cache(hk, context, d)
    for name in ("k", "v"):
        q = np.clip(np.rint(rng.standard_normal(ref.k.shape) * 36), -127, 127).astype(np.int8)
        s = np.exp(rng.standard_normal(ref.ks.shape) * spread) / 36
        setattr(ref, name, q)
        setattr(ref, name + "s", s.astype(np.float32))
    return ref


class Call:
    """One attention_q8_dev call with its buffers."""

    def __init__(self, gpu, rt, q, ref, kend, kstart=None, maxk=None):
        self.gpu, self.q = gpu, q
        T, H, d = q.shape
        hk, C = ref.k.shape[0], ref.context
        raw = gpu.pack_cache_q8(ref.k[:, :C], ref.ks, ref.v[:, :C], ref.vs, ref.bad)
        self.bufs = [dev(rt, a) for a in (q, raw, np.asarray(kend, np.int64), np.asarray(kend if kstart is None else kstart, np.int64))]
        self.out = dev(rt, np.full(q.shape, 7, np.float32))
        maxk = maxk or C
        self.wsb = gpu.attention_q8_workspace_bytes(T, H, hk, d, maxk)
        self.ws = dev(rt, np.full(self.wsb // 4 + 4, np.nan, np.float32))
        self.args = (self.bufs[0].ptr, self.bufs[1].ptr, self.bufs[2].ptr, self.bufs[3].ptr if kstart is not None else None, T, H,
                     hk, d, C, maxk, self.out.ptr, self.ws.ptr, self.wsb)

    def enqueue(self, stream):
        self.gpu.attention_q8_dev(*self.args, stream.handle)

    def result(self):
        return self.out.download(np.float32).reshape(self.q.shape)


def run(gpu, rt, *a, **kw):
    c, s = Call(gpu, rt, *a, **kw), rt.Stream()
    c.enqueue(s)
    s.sync()
    assert np.isnan(c.ws.download(np.float32)[c.wsb // 4:]).all()  # nothing past the workspace
    return c.result()


def check(got, ref, q, kend, kstart=None, maxk=None):
    want, bound = q8_ref.attention(q, *ref.values(), kend, kstart, maxk)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.abs(np.nan_to_num(got) - np.nan_to_num(want))
    assert (off <= np.nan_to_num(bound)[..., None] + 1e-37).all(), (off.max(), np.argwhere(off > bound[..., None])[:5])


# `room`: max_keys, which with T, heads and kv heads decides on the kernels: the
# cache's length, and far more than it (many splits; from 64 tokens the prompt
# kernel beside the other)
@pytest.mark.parametrize("room", [None, 1 << 18])
@pytest.mark.parametrize("T,H,hk,d,slots,stride", [
    (100, 144, 1, 64, 1, 250), (128, 14, 2, 64, 1, 1400), (20, 8, 2, 128, 1, 900), (7, 3, 1, 64, 1, 1500), (33, 4, 4, 192, 1, 700), (2, 16, 2, 256, 1, 4000), (63, 6, 6, 80, 1, 1300), (64, 8, 2, 128, 1, 2500), (109, 14, 2, 128, 3, 260), (97, 34, 1, 64, 2, 150), (260, 8, 8, 128, 1, 900), (120, 3, 1, 256, 1, 400), (1, 1, 1, 64, 1, 32), (1, 4, 1, 8, 1, 1), (1, 32, 8, 64, 1, 181), (2, 16, 16, 128, 2, 33), (3, 14, 2, 64, 3, 500),
    (8, 32, 8, 128, 8, 300), (5, 40, 2, 80, 5, 77), (1, 34, 2, 256, 1, 700), (4, 6, 3, 192, 2, 129), (1, 8, 2, 128, 1, 6000),
    (1, 3, 1, 64, 1, 20001), (64, 4, 2, 64, 16, 70), (70, 14, 2, 64, 7, 90), (200, 32, 8, 128, 1, 200), (133, 8, 8, 64, 1, 300),
    (130, 34, 2, 80, 3, 130), (181, 14, 2, 64, 1, 181), (65, 12, 4, 256, 2, 100), (150, 16, 2, 128, 150, 13), (300, 6, 2, 192, 2, 400)])
def test_attention(gpu, rt, T, H, hk, d, slots, stride, room):
    """Prompts and decode batches, sequences that start inside a block, rows
    that see nothing, keys that no row sees marked as not finite."""
    rng = np.random.default_rng(T * 31 + H + stride)
    C = slots * stride
    ref = random_cache(rng, hk, C, d, spread=0.5)
    q = rng.standard_normal((T, H, d)).astype(np.float32)
    slot = np.sort(np.arange(T) % slots)
    start = slot * stride
    if slots == 1 and T > 1:
        end = np.maximum(C - T, 0) + np.arange(T)
    else:
        end = start + rng.integers(0, stride, T)
        end[-1] = start[-1] + stride - 1
    if T > 2:
        end[T // 3] = start[T // 3] - 1  # sees no key
    used = np.zeros(-(-C // 32) * 32, bool)
    for a, b in zip(start, end):
        used[a:b + 1] = True
    ref.bad[:] = (~used).reshape(-1, 32) @ (1 << np.arange(32, dtype=np.uint64))
    check(run(gpu, rt, q, ref, end, start if slots > 1 else None, room), ref, q, end, start if slots > 1 else None)


@pytest.mark.parametrize("room", [900, 1 << 20])
@pytest.mark.parametrize("H,hk,d", [(4, 1, 64), (8, 8, 128), (14, 2, 64), (3, 1, 192), (16, 2, 256), (10, 2, 8), (36, 2, 128)])
def test_few_rows_of_a_sequence(gpu, rt, H, hk, d, room):
    """Rows that share their keys, as a short prompt's or a draft's: one sequence
    of 20, several of 1 to 5 rows, rows that see nothing, windows, marks."""
    rng = np.random.default_rng(H * d)
    C = 8 * 900
    ref = random_cache(rng, hk, C, d, spread=0.5)
    ref.bad[0, 2 * 900 // 32 + 7] = 5
    for lens in ([20], [1, 5, 3, 4, 2], [2, 2], [7, 1, 1, 1, 1, 1, 1]):
        start = np.concatenate([np.full(n, 900 * i) for i, n in enumerate(lens)])
        end = np.concatenate([900 * i + 880 - 37 * i + np.arange(n) for i, n in enumerate(lens)])
        q = rng.standard_normal((len(end), H, d)).astype(np.float32)
        check(run(gpu, rt, q, ref, end, start, room), ref, q, end, start, room)
        end[-1] = start[-1] - 1
        start[:-1] += rng.integers(0, 40, len(end) - 1)
        check(run(gpu, rt, q, ref, end, start, room), ref, q, end, start, room)


def test_prompts_and_decode_rows_in_one_call(gpu, rt):
    """Tiles of a prompt beside tiles of single rows of many sequences, and tiles
    of both: each row comes from one of the kernels."""
    rng = np.random.default_rng(11)
    for hk, H, d in ((2, 8, 64), (1, 7, 128), (1, 2, 192)):
        stride, singles = 96, 150
        C = stride * singles + 2000
        ref = random_cache(rng, hk, C, d)
        start = [stride * i for i in range(singles)] + [stride * singles] * 333
        end = [s + int(rng.integers(0, stride)) for s in start[:singles]] + [stride * singles + 1500 + i for i in range(333)]
        start, end = np.array(start), np.array(end)
        end[[3, 40, 41, 42, 300]] = start[[3, 40, 41, 42, 300]] - 1
        q = rng.standard_normal((len(end), H, d)).astype(np.float32)
        for room in (2000, 1 << 20):
            check(run(gpu, rt, q, ref, end, start, room), ref, q, end, start, room)


@pytest.mark.parametrize("T", [3, 80, 200])
def test_ranges(gpu, rt, T):
    """Windows anywhere, negative and past the cache, max_keys inside a block."""
    rng = np.random.default_rng(T)
    ref, C = random_cache(rng, 2, 700, 64), 700
    q = rng.standard_normal((T, 8, 64)).astype(np.float32)
    start = rng.integers(-50, C + 40, T)
    end = start + rng.integers(-20, 400, T)
    for maxk in (1, 33, 250, C, 1 << 19):
        check(run(gpu, rt, q, ref, end, start, maxk), ref, q, end, start, maxk)


@pytest.mark.parametrize("T", [1, 100])
@pytest.mark.parametrize("maxk", [256, 4096, 1 << 17])
def test_values_at_the_ends(gpu, rt, T, maxk):
    """Blocks of zeros, value scales from 2^-96 to 1e30 beside each other,
    queries of zeros, tiny, large and with large outliers."""
    rng = np.random.default_rng(T + maxk)
    ref = random_cache(rng, 2, 256, 64)
    ref.vs[:, 1], ref.vs[:, 2], ref.vs[:, 3] = 0, 2.0 ** -96, 1e30
    ref.ks[:, 4], ref.ks[:, 5] = 0, 1e-30
    q = rng.standard_normal((T, 8, 64)).astype(np.float32)
    q[0, 0], q[0, 1], q[0, 2] = 0, q[0, 1] * 1e-30, q[0, 2] * 100
    q[0, 3, 5] = 1000
    q[0, 4] *= 1e-42  # subnormal
    for end in (255, 95, 40, 31):
        kend = np.full(T, end)
        check(run(gpu, rt, q, ref, kend, None, maxk), ref, q, kend)
    only_zeros = np.full(T, 63), np.full(T, 32)
    assert not run(gpu, rt, q, ref, *only_zeros, maxk).any()


@pytest.mark.parametrize("T", [2, 90, 130])
def test_not_finite(gpu, rt, T):
    """A marked entry reaches the rows that see it alone; a query that is not
    finite its own row; scores past float32 give NaN."""
    rng = np.random.default_rng(T)
    ref = random_cache(rng, 1, 300, 128)
    ref.bad[0, 5] = 1 << 7  # entry 167
    q = rng.standard_normal((T, 4, 128)).astype(np.float32)
    kend = np.where(np.arange(T) % 2 == 0, 166, 250)
    check(run(gpu, rt, q, ref, kend), ref, q, kend)
    check(run(gpu, rt, q, ref, kend, None, 1 << 20), ref, q, kend)
    q[0, 1, 3], q[0, 2, 100] = np.nan, np.inf
    got = run(gpu, rt, q, ref, kend)
    assert np.isnan(got[0, 1:3]).all() and np.isfinite(got[0, [0, 3]]).all() and (kend[0] == 166)
    none = np.full(T, -1)
    assert not run(gpu, rt, q, ref, none).any()  # sees nothing: zeros even so
    big = random_cache(rng, 1, 64, 128)
    big.ks[:] = 1e36
    assert np.isnan(run(gpu, rt, np.full((T, 4, 128), 1e10, np.float32), big, np.full(T, 40))).all()


def test_the_most_rows(gpu, rt):
    """65535 rows in one call: a store of as many (a prompt's, then one row a
    block), rope beside it, and attention by either kernel."""
    T, hk, d = 65535, 1, 8
    rng = np.random.default_rng(0)
    for C, index in ((T, np.arange(T)), (32 * T, 32 * np.arange(T) + 5)):
        dc = DeviceCache(gpu, rt, hk, C, d)
        q, k, v = values(rng, T, 2, d), values(rng, T, hk, d), values(rng, T, hk, d)
        dc.store(k, v, index)
        for x, y in zip((k, v), dc.load(index)):  # half a step, of the block's largest / 127, and two roundings
            block = index // 32 - index[0] // 32
            amax = np.zeros(block[-1] + 1)
            np.maximum.at(amax, block, np.abs(x).max((1, 2)))
            assert (np.abs(x.astype(np.float64) - y).max((1, 2)) <= amax[block] / 127 * (0.5 + 127 * 2.0 ** -22)).all()
        one, s = DeviceCache(gpu, rt, hk, C, d), rt.Stream()
        pos, freq = np.zeros(T, np.int64), np.array([1.0, 0.5])
        b = [dev(rt, a) for a in (q, k, v, pos, index.astype(np.int64), freq)]
        gpu.rope_kv_q8_dev(*(x.ptr for x in b), T, 2, hk, d, 4, 1, C, one.buf.ptr, s.handle)  # (an angle of 0)
        s.sync()
        assert np.array_equal(one.raw(), dc.raw()) and np.array_equal(b[0].download(np.float32).reshape(q.shape), q)
    small = random_cache(rng, hk, 300, d)
    end = rng.integers(-1, 300, T)
    some = np.concatenate([[0, 1, 32767, 65533, 65534], rng.integers(0, T, 300)])
    for room in (32, 64, 300, 1 << 20):
        got = run(gpu, rt, q, small, end, None, room)
        check(got[some], small, q[some], end[some], None, room)


@pytest.mark.parametrize("T,room", [(1, 1 << 16), (8, 3000), (200, 1 << 18)])
def test_the_same_bits_every_time(gpu, rt, T, room):
    """Nothing depends on the order of workgroups: two calls at once on two
    streams, each with its workspace, give one call's bits; so does a call with
    other rows beside these where the cut is the same."""
    rng = np.random.default_rng(T)
    ref = random_cache(rng, 2, 3000, 64)
    q = rng.standard_normal((T, 8, 64)).astype(np.float32)
    kend = 2999 - np.arange(T)[::-1]
    want = run(gpu, rt, q, ref, kend, None, room)
    calls = [Call(gpu, rt, q, ref, kend, None, room) for _ in range(2)]
    streams = [rt.Stream(), rt.Stream()]
    for _ in range(3):
        for c, s in zip(calls, streams):
            c.enqueue(s)
        for c, s in zip(calls, streams):
            s.sync()
            assert np.array_equal(c.result(), want)


def test_graphs_share_a_workspace(gpu, rt):
    """Two captured calls with one workspace, replayed in turn with other
    calls between, on another stream too: the eager bits every time."""
    rng = np.random.default_rng(5)
    ref = random_cache(rng, 2, 3000, 64)
    calls = []
    for T in (1, 3):
        q = rng.standard_normal((T, 8, 64)).astype(np.float32)
        calls.append(Call(gpu, rt, q, ref, np.array([2999, 1500, 40])[:T]))
        assert calls[-1].wsb > 0
    big = max(calls, key=lambda c: c.wsb)
    s, s2 = rt.Stream(), rt.Stream()
    want, graphs = [], []
    for c in calls:
        c.args = c.args[:-2] + (big.ws.ptr, big.wsb)
        c.enqueue(s)
        s.sync()
        want.append(c.result())
        check(want[-1], ref, c.q, np.array([2999, 1500, 40])[:len(c.q)])
        graphs.append(rt.Graph(s, lambda c=c: c.enqueue(s)))
    for i in range(6):
        for c, g, w in zip(calls, graphs, want):
            c.out.zero()
            g.launch(s if i % 2 else s2)
            (s if i % 2 else s2).sync()
            assert np.array_equal(c.result(), w)
            c.enqueue(s2)
            s2.sync()
            assert np.array_equal(c.result(), w)


@pytest.mark.parametrize("T,H,hk", [(1, 4, 1), (6, 8, 2), (40, 4, 1), (100, 8, 4), (130, 14, 2)])
def test_a_graph_over_growing_keys(gpu, rt, T, H, hk):
    """One captured call, replayed with the rows' keys changed: more and fewer,
    one sequence and many, none; what an earlier replay left in the workspace
    does not matter."""
    rng = np.random.default_rng(T)
    C, room = 6000, 1 << 17
    ref = random_cache(rng, hk, C, 64)
    q = rng.standard_normal((T, H, 64)).astype(np.float32)
    c, s = Call(gpu, rt, q, ref, np.zeros(T), np.zeros(T), room), rt.Stream()
    g = rt.Graph(s, lambda: c.enqueue(s))
    for n in (5, 5999, 40, 256, 2000, 257, -1, 600, 4100):
        for spread in (False, True):
            start = rng.integers(0, C, T) if spread else np.zeros(T, np.int64)
            end = start + rng.integers(-1, max(n, 1), T) if spread else np.maximum(n - T, -1) + np.arange(T)
            c.bufs[2].upload(end.astype(np.int64))
            c.bufs[3].upload(start.astype(np.int64))
            g.launch(s)
            s.sync()
            got = c.result()
            c.enqueue(s)
            s.sync()
            assert np.array_equal(got, c.result(), equal_nan=True)
            some = rng.integers(0, T, 12)
            check(got[some], ref, q[some], end[some], start[some], room)


def test_offsets_past_32_bits(gpu, rt):
    """The last blocks of a cache whose bytes pass 2^32: stored, read back and
    attended to."""
    hk, d, C = 1, 256, 9_000_000  # 4.6 GB
    dc = DeviceCache(gpu, rt, hk, C, d)
    assert dc.buf.nbytes > 1 << 32
    rng = np.random.default_rng(0)
    T = 70
    index = C - T + np.arange(T)
    k, v = values(rng, T, hk, d), values(rng, T, hk, d)
    dc.store(k, v, index)
    base = (C - T) // 32 * 32
    ref = q8_ref.Cache(hk, C - base, d)
    ref.store(k, v, index - base)
    got = dc.load(index)
    lo = C - T - base
    for g, w in zip(got, ref.values()):
        assert np.array_equal(g[:, 0], w[0, lo:].astype(np.float32))
    q = rng.standard_normal((T, 2, d)).astype(np.float32)
    bufs = [dev(rt, a) for a in (q, index, np.full(T, C - T))]
    out = rt.DeviceBuffer(q.nbytes)
    wsb = gpu.attention_q8_workspace_bytes(T, 2, hk, d, 100)
    ws = rt.DeviceBuffer(wsb)
    gpu.attention_q8_dev(bufs[0].ptr, dc.buf.ptr, bufs[1].ptr, bufs[2].ptr, T, 2, hk, d, C, 100, out.ptr, ws.ptr, wsb, dc.s.handle)
    dc.s.sync()
    check(out.download(np.float32).reshape(q.shape), ref, q, index - base, np.full(T, lo), 100)
