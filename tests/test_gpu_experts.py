"""The operators of a mixture of experts (experts_route.hip, experts.hip)
against their float64 restatement, and the products bit for bit against the
oracle's product with each expert's own matrix."""
import numpy as np
import pytest

import experts_ref as ref

pytestmark = pytest.mark.gpu
Q8_0, Q4_K, Q6_K = 64, 66, 67


@pytest.fixture(scope="module")
def rt(gpu):
    import hiprt

    return hiprt


class Guarded:
    """A device buffer with a pattern behind it that must stay."""

    def __init__(self, rt, nbytes, fill=7):
        self.nbytes = nbytes
        self.b = rt.DeviceBuffer.from_array(np.full(nbytes + 256, fill, np.uint8))
        self.ptr = self.b.ptr

    def read(self, dtype, shape):
        a = self.b.download(np.uint8)
        assert (a[self.nbytes:] == 7).all()
        return a[:self.nbytes].view(dtype)[:int(np.prod(shape))].reshape(shape)


def plan_of(gpu, rt, ids, experts):
    T, top = ids.shape
    s, nb = rt.Stream(), gpu.experts_plan_bytes(T, top, experts)
    dev, out = rt.DeviceBuffer.from_array(ids.astype(np.int32)), Guarded(rt, nb)
    gpu.experts_plan_dev(dev.ptr, T, top, experts, out.ptr, nb, s.handle)
    s.sync()
    return out.read(np.int32, (nb // 4,))


def same_plan(got, ids, experts):
    want, pairs = ref.packed_plan(ids, experts), ids.size
    up = lambda n: (n + 63) // 64 * 64  # noqa: E731
    at = up(experts + 1)
    for a, b in ((0, experts + 1), (at, at + pairs), (at + up(pairs), at + up(pairs) + pairs)):
        np.testing.assert_array_equal(got[a:b], want[a:b])


@pytest.mark.parametrize("T,top,experts", [(1, 1, 1), (1, 2, 8), (3, 8, 64), (64, 1, 7), (65, 2, 60), (181, 4, 60), (1000, 8, 128),
                                           (1025, 1, 512), (2048, 8, 256), (70001, 2, 5),
                                           (4096, 1, 3), (4097, 1, 3), (5461, 3, 64), (16385, 1, 2)])
def test_plan(gpu, rt, T, top, experts):
    ids = np.random.default_rng(T * 7 + experts).integers(0, experts, (T, top))
    same_plan(plan_of(gpu, rt, ids, experts), ids, experts)


@pytest.mark.parametrize("what", ["none", "one", "padded", "outside"])
def test_plan_uneven(gpu, rt, what):
    r = np.random.default_rng(3)
    ids = r.integers(0, 9, (300, 3))
    if what == "none":
        ids[:] = -1
    elif what == "one":
        ids[:] = 8
    elif what == "padded":
        ids[211:] = -1
        ids[5, 1] = -1
    else:
        ids[::7] = 9
        ids[::11, 0] = 2 ** 31 - 1
        ids[::13, 1] = -2 ** 31
    same_plan(plan_of(gpu, rt, ids, 9), ids, 9)


def test_plan_of_no_tokens(gpu, rt):
    s, nb = rt.Stream(), gpu.experts_plan_bytes(0, 2, 8)
    out = Guarded(rt, nb)
    gpu.experts_plan_dev(None, 0, 2, 8, out.ptr, nb, s.handle)
    s.sync()
    assert (out.read(np.int32, (nb // 4,))[:9] == 0).all()


def run_route(gpu, rt, x, router, top, normalize, with_plan=True):
    (T, k), experts = x.shape, router.shape[0]
    s, nb, wsb = rt.Stream(), gpu.experts_plan_bytes(T, top, experts), gpu.experts_route_workspace_bytes(T, experts)
    dx, dr = rt.DeviceBuffer.from_array(x), rt.DeviceBuffer.from_array(router)
    ids, w, plan, ws = Guarded(rt, T * top * 4), Guarded(rt, T * top * 4), Guarded(rt, nb), Guarded(rt, wsb)
    gpu.experts_route_dev(dx.ptr, dr.ptr, T, k, experts, top, normalize, ids.ptr, w.ptr, plan.ptr if with_plan else None, nb, ws.ptr,
                          wsb, s.handle)
    s.sync()
    ws.read(np.uint8, (1,))
    got = plan.read(np.int32, (nb // 4,))
    if with_plan:
        same_plan(got, ids.read(np.int32, (T, top)), experts)
    else:
        assert (got.view(np.uint8) == 7).all()
    return ids.read(np.int32, (T, top)), w.read(np.float32, (T, top))


def check_route(got, x, router, top, normalize):
    ids, w = ref.route(x, router, top, normalize)
    np.testing.assert_array_equal(got[0], ids)
    np.testing.assert_array_equal(np.isnan(got[1]), np.isnan(w))
    # in float64 up to the last rounding, with a 2^-20 part of it for the rest
    fine = ~np.isnan(w)
    assert (np.abs(got[1][fine] - w[fine]) <= (1 + 2.0 ** -20) * ref.EPS * w[fine] + 2.0 ** -150).all()


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("T,k,experts,top", [(1, 4096, 8, 2), (1, 4, 1, 1), (1, 20, 3, 3), (3, 2048, 64, 8), (16, 516, 60, 4),
                                             (17, 1000, 17, 1), (181, 2048, 60, 4), (37, 256, 512, 32), (50, 64, 200, 7),
                                             (33, 4100, 128, 8), (300, 132, 65, 5), (700, 260, 200, 6),
                                             (32, 512, 40, 16), (1030, 68, 130, 3),
                                             (4, 256, 32, 32), (3, 1364, 8, 2), (2, 12, 512, 5), (1, 2052, 15, 4)])
def test_route(gpu, rt, T, k, experts, top, normalize):
    r = np.random.default_rng(T + 10 * k + experts)
    x, router = r.standard_normal((T, k), np.float32), (r.standard_normal((experts, k)) / np.sqrt(k) * 1.5).astype(np.float32)
    check_route(run_route(gpu, rt, x, router, top, normalize, with_plan=T != 17), x, router, top, normalize)


def test_route_equal_logits_go_by_the_index(gpu, rt):
    r = np.random.default_rng(5)
    x, router = r.standard_normal((40, 256), np.float32), r.standard_normal((70, 256), np.float32) / 16
    router[[3, 19, 40, 69]] = router[11]
    router[50:60] = router[5]
    x[7] = 0
    check_route(run_route(gpu, rt, x, router, 12, True), x, router, 12, True)


# a token a wave of one workgroup, a plan of more than 64 pairs there; parts of K
# that do not fill the loads of eight; the lower halves of equal upper ones
@pytest.mark.parametrize("T,k,experts,top", [(16, 2300, 32, 20), (16, 4096, 32, 4), (8, 3000, 64, 32), (5, 4096, 100, 9), (17, 2048, 30, 6),
                                             (600, 1040, 8, 2), (64, 1024, 300, 3)])
def test_route_in_parts(gpu, rt, T, k, experts, top):
    r = np.random.default_rng(T + k)
    x, router = r.standard_normal((T, k), np.float32), (r.standard_normal((experts, k)) / np.sqrt(k)).astype(np.float32)
    check_route(run_route(gpu, rt, x, router, top, True), x, router, top, True)


@pytest.mark.parametrize("T,experts", [(2, 70), (40, 70), (40, 200), (40, 500)])
def test_route_equal_and_close_logits(gpu, rt, T, experts):
    """Logits 1 + 2^-40 i, exact sums of two products: equal upper halves in
    many lanes and slots; every third one equal to the one before it."""
    x = np.zeros((T, 4), np.float32)
    x[:, 0], x[:, 1] = 1, 2.0 ** -40
    x[1] *= -1
    router = np.zeros((experts, 4), np.float32)
    router[:, 0] = 1
    router[:, 1] = np.random.default_rng(experts).permutation(experts)
    router[2::3, 1] = router[1::3, 1][:len(router[2::3])]
    check_route(run_route(gpu, rt, x, router, 20, True), x, router, 20, True)


@pytest.mark.parametrize("experts", [9, 100])
def test_route_of_values_that_are_not_finite(gpu, rt, experts):
    r = np.random.default_rng(6)
    x, router = r.standard_normal((30, 64), np.float32), r.standard_normal((experts, 64), np.float32)
    x[3, 5], x[4, 60], x[5, 0] = np.nan, np.inf, -np.inf
    router[2, 7] = np.nan
    router[4, 9], router[6, 9] = np.inf, -np.inf
    for normalize in (True, False):
        check_route(run_route(gpu, rt, x, router, 5, normalize), x, router, 5, normalize)


# ---- the products --------------------------------------------------------------------

class Layer:
    """Weights of `experts` experts, their bytes on the host too."""

    def __init__(self, gpu, oracle, dt, experts, n, k, seed, edit=None):
        self.dt, self.experts, self.n, self.k = dt, experts, n, k
        self.raw = oracle.synthetic_weight(dt, experts * n, k, seed=seed, scale=1 / np.sqrt(k)).reshape(experts, -1)
        if edit:
            edit(self.raw)
        self.w = gpu.Weight(self.raw.reshape(-1), dt, experts * n, k)


def choices(seed, T, top, experts, what="even"):
    r = np.random.default_rng(seed)
    ids = np.stack([r.permutation(max(experts, top))[:top] for _ in range(T)])
    if what == "one":  # all tokens to the same experts
        ids[:] = np.arange(top) + (experts - top)
    elif what == "padded":
        ids[T - T // 3:] = -1
        ids[::5, 0] = -1
    elif what == "again":  # the same expert twice for a token
        ids[:, -1] = ids[:, 0]
    elif what == "none":
        ids[:] = -1
    return ids.astype(np.int32)


def run_swiglu(gpu, rt, gate, up, x, ids, stream=None):
    (T, k), top, n = x.shape, ids.shape[1], gate.n
    plan = rt.DeviceBuffer.from_array(ref.packed_plan(ids, gate.experts))
    wsb = gpu.experts_swiglu_workspace_bytes(T, top, n, k)
    dx, h, ws, s = rt.DeviceBuffer.from_array(x), Guarded(rt, T * top * n * 4), Guarded(rt, wsb), stream or rt.Stream()
    gpu.experts_swiglu_a8_dev(gate.w, up.w, gate.experts, dx.ptr, T, top, plan.ptr, plan.nbytes, h.ptr, ws.ptr, wsb, s.handle)
    s.sync()
    ws.read(np.uint8, (1,))
    return h.read(np.float32, (T * top, n))


def run_combine(gpu, rt, down, h, weights, ids):
    T, top = ids.shape
    plan = rt.DeviceBuffer.from_array(ref.packed_plan(ids, down.experts))
    wsb = gpu.experts_combine_workspace_bytes(T, top, down.n, down.k)
    dh, dw = rt.DeviceBuffer.from_array(h), rt.DeviceBuffer.from_array(weights)
    y, ws, s = Guarded(rt, T * down.n * 4), Guarded(rt, wsb), rt.Stream()
    gpu.experts_combine_a8_dev(down.w, down.experts, dh.ptr, dw.ptr, T, top, plan.ptr, plan.nbytes, y.ptr, ws.ptr, wsb, s.handle)
    s.sync()
    ws.read(np.uint8, (1,))
    return y.read(np.float32, (T, down.n))


def bits(a):
    return np.ascontiguousarray(a, np.float32).view(np.uint32)


def expert_products(oracle, layer, x, ids, exact):
    """Each pair's product with its row of x: bit for bit (K-quants) or (values, bounds)."""
    flat = ids.reshape(-1)
    y, b = np.zeros((flat.size, layer.n)), np.zeros((flat.size, layer.n))
    for e in range(layer.experts):
        at = np.nonzero(flat == e)[0]
        if at.size == 0:
            continue
        if exact:
            y[at] = oracle.linear_a8(x[at], layer.raw[e], layer.dt, layer.n, layer.k, block=256, threads=8)
        else:
            y[at], b[at] = ref.product(x[at], layer.raw[e], layer.dt, layer.n, layer.k)
    return (y.astype(np.float32) if exact else y), b


def check_swiglu(got, oracle, gate, up, x, ids):
    has = ids.reshape(-1) >= 0
    assert (bits(got[~has]) == 0x07070707).all()  # left as they were
    xs = np.repeat(x, ids.shape[1], 0)
    if gate.dt != Q8_0:
        g, u = (expert_products(oracle, w, xs, ids, True)[0][has] for w in (gate, up))
        pad = -g.size % 8
        want = oracle.silu_mul(np.append(g, np.zeros(pad, np.float32)), np.append(u, np.zeros(pad, np.float32)), 1)
        np.testing.assert_array_equal(bits(got[has]), bits(want[:g.size].reshape(g.shape)))
    (g, ge), (u, ue) = (expert_products(oracle, w, xs, ids, False) for w in (gate, up))
    want, bound = ref.swiglu(g, ge, u, ue)
    assert (np.abs(got[has] - want[has]) <= bound[has]).all()


def check_combine(got, oracle, down, h, weights, ids):
    T, top = ids.shape
    y, b = expert_products(oracle, down, h, ids, False)
    w = weights.astype(np.float64)[..., None] * (ids >= 0)[..., None]
    y, b = y.reshape(T, top, -1), b.reshape(T, top, -1)
    # top fmas, each EPS of the sum so far
    bound = (np.abs(w) * b).sum(1) * (1 + 2 * top * ref.EPS) + 1.01 * top * ref.EPS * (np.abs(w) * (np.abs(y) + b)).sum(1)
    assert (np.abs(got - (w * y).sum(1)) <= bound).all()
    assert (bits(got[(ids < 0).all(1)]) == 0).all()


SHAPES = [  # dt, experts, n, k, T, top, choices
    (Q4_K, 8, 128, 512, 1, 2, "even"), (Q4_K, 8, 96, 256, 1, 1, "even"), (Q4_K, 4, 70, 768, 5, 2, "even"),
    (Q4_K, 3, 33, 1280, 40, 2, "even"), (Q4_K, 60, 64, 512, 33, 4, "padded"), (Q4_K, 5, 129, 512, 200, 3, "one"),
    (Q4_K, 130, 32, 256, 7, 8, "even"), (Q4_K, 2, 256, 512, 300, 2, "again"), (Q4_K, 6, 64, 256, 9, 2, "none"),
    (Q4_K, 1, 1, 256, 65, 1, "even"),
    (Q6_K, 8, 128, 512, 1, 2, "even"), (Q6_K, 8, 97, 256, 1, 1, "even"), (Q6_K, 4, 70, 768, 5, 2, "padded"),
    (Q6_K, 3, 35, 1280, 40, 2, "even"), (Q6_K, 60, 64, 256, 33, 4, "even"), (Q6_K, 5, 129, 512, 200, 3, "one"),
    (Q6_K, 2, 256, 512, 300, 2, "again"), (Q6_K, 512, 2, 256, 12, 4, "even"),
    (Q8_0, 8, 128, 512, 1, 2, "even"), (Q8_0, 8, 97, 32, 1, 1, "even"), (Q8_0, 4, 70, 736, 5, 2, "even"),
    (Q8_0, 3, 35, 1312, 40, 2, "padded"), (Q8_0, 60, 64, 96, 33, 4, "even"), (Q8_0, 5, 129, 544, 200, 3, "one"),
    (Q8_0, 2, 256, 512, 300, 2, "again"), (Q8_0, 6, 64, 224, 9, 2, "none"),
    # few pairs, some without an expert or with one twice; too many choices or
    # blocks for one workgroup's table
    (Q4_K, 8, 64, 512, 3, 2, "padded"), (Q4_K, 8, 63, 1024, 4, 2, "again"), (Q4_K, 64, 20, 256, 2, 8, "none"),
    (Q4_K, 64, 8, 8192, 2, 32, "even"), (Q6_K, 8, 64, 512, 3, 2, "padded"), (Q6_K, 8, 63, 1024, 4, 2, "again"),
    (Q6_K, 40, 33, 768, 5, 8, "padded"), (Q8_0, 8, 64, 512, 3, 2, "padded"), (Q8_0, 8, 63, 1056, 2, 2, "again"),
    (Q8_0, 64, 20, 96, 2, 8, "none"), (Q8_0, 16, 9, 8192, 1, 8, "even"), (Q8_0, 40, 33, 800, 5, 8, "padded"),
    # long rows (whole turns of the slots), tiles of 32 and of 64 and 96 pairs
    (Q4_K, 3, 64, 2560, 30, 2, "even"), (Q4_K, 2, 40, 4352, 70, 1, "padded"), (Q4_K, 1, 66, 4864, 80, 1, "even"),
    (Q6_K, 3, 64, 2560, 30, 2, "even"), (Q6_K, 1, 130, 2304, 100, 1, "even"), (Q6_K, 2, 33, 4352, 190, 2, "one"),
    (Q8_0, 3, 64, 2560, 30, 2, "even"), (Q8_0, 1, 66, 2336, 80, 1, "even"), (Q8_0, 2, 65, 2304, 190, 2, "padded"),
]


def acts_for(seed, rows, k):
    x = np.random.default_rng(seed).standard_normal((rows, k), np.float32)
    x[:, 3::37] *= 4
    x[rows // 2, : k // 2] = 0
    return x


@pytest.mark.parametrize("dt,experts,n,k,T,top,what", SHAPES)
def test_swiglu(gpu, rt, oracle, dt, experts, n, k, T, top, what):
    gate, up = (Layer(gpu, oracle, dt, experts, n, k, seed) for seed in (1, 2))
    x, ids = acts_for(3, T, k), choices(4, T, top, experts, what)
    check_swiglu(run_swiglu(gpu, rt, gate, up, x, ids), oracle, gate, up, x, ids)


@pytest.mark.parametrize("dt,experts,n,k,T,top,what", SHAPES)
def test_combine(gpu, rt, oracle, dt, experts, n, k, T, top, what):
    down = Layer(gpu, oracle, dt, experts, n, k, 5)
    h, ids = acts_for(6, T * top, k), choices(7, T, top, experts, what)
    weights = np.random.default_rng(8).random((T, top), np.float32)
    check_combine(run_combine(gpu, rt, down, h, weights, ids), oracle, down, h, weights, ids)


# tiles of 64 pairs of which the last one has all, more than half, few
TILES = [(dt, 2, 97, 768, T, 1, what) for dt in (Q4_K, Q6_K, Q8_0) for T, what in ((128, "even"), (180, "one"), (150, "even"), (130, "one"))]


@pytest.mark.parametrize("dt,experts,n,k,T,top,what", TILES)
def test_last_tiles(gpu, rt, oracle, dt, experts, n, k, T, top, what):
    test_swiglu(gpu, rt, oracle, dt, experts, n, k, T, top, what)
    test_combine(gpu, rt, oracle, dt, experts, n, k, T, top, what)


# tiles of 32 and of 16 weight rows a wave where the other ones of these sizes run
GRIDS = [(Q4_K, 60, 530, 512, 33, 4, "padded"), (Q4_K, 9, 200, 1280, 60, 2, "even"), (Q4_K, 3, 65, 4864, 40, 1, "even"),
         (Q6_K, 20, 1730, 2304, 150, 4, "padded"), (Q6_K, 60, 70, 2048, 90, 4, "even"), (Q6_K, 3, 79, 4864, 40, 1, "even")]


@pytest.mark.parametrize("dt,experts,n,k,T,top,what", GRIDS)
def test_rows_of_a_wave(gpu, rt, oracle, dt, experts, n, k, T, top, what):
    test_combine(gpu, rt, oracle, dt, experts, n, k, T, top, what)


# pairs each by itself where there are many more experts, and just above
MANY = [(dt, experts, n, k, T, 8, what) for dt in (Q4_K, Q6_K) for experts, n, k, T, what in (
    (128, 24, 512, 3, "even"), (200, 16, 4096, 6, "padded"), (200, 16, 4096, 7, "even"), (128, 12, 256, 12, "again"),
    (130, 12, 512, 16, "padded"), (130, 12, 256, 17, "even"))]


@pytest.mark.parametrize("dt,experts,n,k,T,top,what", MANY)
def test_pairs_of_many_experts(gpu, rt, oracle, dt, experts, n, k, T, top, what):
    test_swiglu(gpu, rt, oracle, dt, experts, n, k, T, top, what)
    test_combine(gpu, rt, oracle, dt, experts, n, k, T, top, what)


@pytest.mark.parametrize("dt", [Q4_K, Q6_K])
@pytest.mark.parametrize("T", [1, 3, 50, 200])
def test_products_equal_the_oracle_bit_for_bit(gpu, rt, oracle, dt, T):
    """One choice of weight one: y is the product itself."""
    down = Layer(gpu, oracle, dt, 3, 131, 1024, 9)
    h, ids = acts_for(10, T, 1024), choices(11, T, 1, 3)
    got = run_combine(gpu, rt, down, h, np.ones((T, 1), np.float32), ids)
    np.testing.assert_array_equal(bits(got), bits(expert_products(oracle, down, h, ids, True)[0]))


def test_q8_0_products_equal_the_tiled_ones_bit_for_bit(gpu, rt, oracle):
    down = Layer(gpu, oracle, Q8_0, 2, 256, 512, 12)
    h, ids = acts_for(13, 128, 512), choices(14, 128, 1, 2)
    got = run_combine(gpu, rt, down, h, np.ones((128, 1), np.float32), ids)
    s, wsb = rt.Stream(), gpu.a8_workspace_bytes(128, 512)
    dh, ws, y = rt.DeviceBuffer.from_array(h), rt.DeviceBuffer(wsb), rt.DeviceBuffer(128 * 256 * 4)
    for e in range(2):
        w = gpu.Weight(down.raw[e], Q8_0, 256, 512)
        gpu.quantize_act_dev(dh.ptr, 128, 512, 32, ws.ptr, wsb, s.handle)
        gpu.matmul_a8_quantized_q8_0_tiled_dev(w, dh.ptr, 128, None, y.ptr, ws.ptr, wsb, s.handle)
        s.sync()
        want = y.download(np.float32).reshape(128, 256)
        at = ids[:, 0] == e
        np.testing.assert_array_equal(bits(got[at]), bits(want[at]))


@pytest.mark.parametrize("dt", [Q4_K, Q6_K, Q8_0])
@pytest.mark.parametrize("T", [2, 70])
def test_refused_rows_take_the_float32_path(gpu, rt, oracle, dt, T):
    """Rows of x with NaN or beyond 2^60 and weight rows with a scale that is
    not finite: as linear_a8 has them, and no other row sees them."""
    nb, off = {Q4_K: (144, 0), Q6_K: (210, 208), Q8_0: (34, 0)}[dt]

    def edit(raw):
        b = raw.reshape(3, 70, -1, nb)
        b[1, 7, 0, off:off + 2] = [0, 0x7C]     # inf
        b[2, 69, -1, off:off + 2] = [1, 0x7E]   # NaN

    gate, up = Layer(gpu, oracle, dt, 3, 70, 512, 15, edit), Layer(gpu, oracle, dt, 3, 70, 512, 16)
    x, ids = acts_for(17, T, 512), choices(18, T, 2, 3)
    x[1, 9] = np.nan
    x[0, 500] = 2.0 ** 61
    got = run_swiglu(gpu, rt, gate, up, x, ids)
    plain = x.copy()
    plain[:2] = acts_for(19, 2, 512)
    fine = run_swiglu(gpu, rt, gate, up, plain, ids)
    np.testing.assert_array_equal(bits(got[4:]), bits(fine[4:]))  # (pairs of the other tokens)
    block = 32 if dt == Q8_0 else 256
    with np.errstate(all="ignore"):
        for p in range(min(T, 6) * 2):
            e, t = ids.reshape(-1)[p], p // 2
            g, u = (oracle.linear_a8(x[t:t + 1], w.raw[e], dt, 70, 512, block=block)[0] for w in (gate, up))
            if dt == Q8_0:  # another order where nothing is refused
                rows = [7] if e == 1 else [69] if e == 2 else []
                rows = np.arange(70) if t < 2 else np.array(rows, int)
            else:
                rows = np.arange(70)
            pad = np.zeros(8 - 70 % 8, np.float32)
            want = oracle.silu_mul(np.append(g, pad), np.append(u, pad), 1)[:70]
            a, b = got[p][rows], want[rows]
            if dt == Q8_0:  # up is in the tiled order where gate alone is refused
                np.testing.assert_array_equal(np.isnan(a), np.isnan(b))
                ok = np.isfinite(b) & (np.abs(b) > 1e-6)
                assert (np.abs(a[ok] - b[ok]) <= 64 * ref.EPS * 512 * np.abs(b[ok])).all()
            else:
                np.testing.assert_array_equal(np.isnan(a), np.isnan(b))
                np.testing.assert_array_equal(bits(a[~np.isnan(a)]), bits(b[~np.isnan(b)]))


def test_a_pair_does_not_depend_on_the_others(gpu, rt, oracle):
    gate, up = (Layer(gpu, oracle, Q4_K, 4, 64, 512, seed) for seed in (20, 21))
    x, ids = acts_for(22, 300, 512), choices(23, 300, 2, 4)
    many = run_swiglu(gpu, rt, gate, up, x, ids).reshape(300, 2, 64)
    for t in (0, 7, 299):
        np.testing.assert_array_equal(bits(run_swiglu(gpu, rt, gate, up, x[t:t + 1], ids[t:t + 1])), bits(many[t]))


def test_two_streams_with_workspaces_of_their_own(gpu, rt, oracle):
    """Calls under way at the same time on two streams, equal bits each time."""
    gate, up = (Layer(gpu, oracle, Q4_K, 6, 128, 1024, seed) for seed in (50, 51))
    B, streams, runs = rt.DeviceBuffer, [rt.Stream(), rt.Stream()], []
    for i, s in enumerate(streams):
        T = (90, 3)[i]
        x, ids = acts_for(52 + i, T, 1024), choices(54 + i, T, 2, 6)
        want = run_swiglu(gpu, rt, gate, up, x, ids)
        plan, dx, h = B.from_array(ref.packed_plan(ids, 6)), B.from_array(x), B(T * 2 * 128 * 4)
        wsb = gpu.experts_swiglu_workspace_bytes(T, 2, 128, 1024)
        runs.append((T, plan, dx, h, B(wsb), wsb, s, want))
    for _ in range(5):
        for T, plan, dx, h, ws, wsb, s, _w in runs:
            gpu.experts_swiglu_a8_dev(gate.w, up.w, 6, dx.ptr, T, 2, plan.ptr, plan.nbytes, h.ptr, ws.ptr, wsb, s.handle)
    for T, plan, dx, h, ws, wsb, s, want in runs:
        s.sync()
        np.testing.assert_array_equal(bits(h.download(np.float32).reshape(T * 2, 128)), bits(want))


def test_a_layer_captured_and_replayed(gpu, rt, oracle):
    """Router, plan, gate and up, down and the sum in one graph, over changing
    inputs, against the eager calls."""
    T, top, E, k, n = 12, 2, 8, 512, 256
    gate, up, down = Layer(gpu, oracle, Q4_K, E, n, k, 24), Layer(gpu, oracle, Q4_K, E, n, k, 25), Layer(gpu, oracle, Q6_K, E, k, n, 26)
    router = np.random.default_rng(27).standard_normal((E, k), np.float32) / 16
    B, s = rt.DeviceBuffer, rt.Stream()
    dr, x, ids, w = B.from_array(router), B(T * k * 4), B(T * top * 4), B(T * top * 4)
    nb = gpu.experts_plan_bytes(T, top, E)
    wsb = max(gpu.experts_route_workspace_bytes(T, E), gpu.experts_swiglu_workspace_bytes(T, top, n, k),
              gpu.experts_combine_workspace_bytes(T, top, k, n))
    plan, h, ws = B(nb), B(T * top * n * 4), B(wsb)

    def enqueue(y):
        gpu.experts_route_dev(x.ptr, dr.ptr, T, k, E, top, True, ids.ptr, w.ptr, plan.ptr, nb, ws.ptr, wsb, s.handle)
        gpu.experts_swiglu_a8_dev(gate.w, up.w, E, x.ptr, T, top, plan.ptr, nb, h.ptr, ws.ptr, wsb, s.handle)
        gpu.experts_combine_a8_dev(down.w, E, h.ptr, w.ptr, T, top, plan.ptr, nb, y.ptr, ws.ptr, wsb, s.handle)

    y, eager = B(T * k * 4), B(T * k * 4)
    x.upload(acts_for(28, T, k))
    enqueue(eager)
    s.sync()
    g = rt.Graph(s, lambda: enqueue(y))
    for seed in range(4):
        xs = acts_for(30 + seed, T, k)
        x.upload(xs)
        g.launch(s)
        s.sync()
        got = y.download(np.float32).reshape(T, k)
        choice, weights = ids.download(np.int32).reshape(T, top), w.download(np.float32).reshape(T, top)
        check_route((choice, weights), xs, router, top, True)
        hs = h.download(np.float32).reshape(T * top, n)
        check_swiglu(hs, oracle, gate, up, xs, choice)
        check_combine(got, oracle, down, hs, weights, choice)
        enqueue(eager)
        s.sync()
        np.testing.assert_array_equal(bits(got), bits(eager.download(np.float32).reshape(T, k)))
    g.destroy()


@pytest.mark.parametrize("dt,T,experts,n,k", [(dt, T, 3, 70, 512) for dt in (Q4_K, Q6_K, Q8_0) for T in (2, 70, 220)] +
                         [(Q4_K, 100, 60, 520, 512), (Q6_K, 100, 60, 1154, 2304)])
def test_refused_rows_of_the_sum(gpu, rt, oracle, dt, T, experts, n, k):
    """The same for down, one choice of weight one."""
    nb, off = {Q4_K: (144, 0), Q6_K: (210, 208), Q8_0: (34, 0)}[dt]

    def edit(raw):
        b = raw.reshape(experts, n, -1, nb)
        b[1, 7, 0, off:off + 2] = [0, 0x7C]
        b[2, n - 1, -1, off:off + 2] = [1, 0x7E]

    down = Layer(gpu, oracle, dt, experts, n, k, 75, edit)
    h, ids = acts_for(76, T, k), choices(77, T, 1, experts)
    ids[:4, 0] = [0, 1, 2, 1][:T]
    h[1, 9] = np.nan
    h[0, k - 12] = 2.0 ** 61
    got = run_combine(gpu, rt, down, h, np.ones((T, 1), np.float32), ids)
    with np.errstate(all="ignore"):
        for t in [*range(min(T, 6)), *range(6, T, 9)]:
            e = ids[t, 0]
            want = oracle.linear_a8(h[t:t + 1], down.raw[e], dt, n, k, block=32 if dt == Q8_0 else 256)[0]
            np.testing.assert_array_equal(np.isnan(got[t]), np.isnan(want))
            fine = ~np.isnan(want)
            if dt == Q8_0:  # (its tiles' order)
                fine &= np.isfinite(want)
                assert (np.abs(got[t] - want)[fine] <= 8 * k * ref.EPS * np.abs(want[fine]).max(initial=0)).all()
            else:
                np.testing.assert_array_equal(bits(got[t][fine]), bits(want[fine]))


class View:
    """Bytes of a weights section from `offset` on, as a layer."""

    def __init__(self, section, offset, dt, experts, n, k, nbytes):
        self.dt, self.experts, self.n, self.k = dt, experts, n, k
        self.w = section.view(offset, nbytes, dt, experts * n, k)


@pytest.mark.parametrize("dt,offset", [(Q4_K, 16), (Q4_K, 208), (Q6_K, 2), (Q6_K, 62), (Q8_0, 2), (Q8_0, 4), (Q8_0, 94)])
@pytest.mark.parametrize("T", [2, 40, 300])
def test_weights_at_the_alignment_of_their_blocks(gpu, rt, oracle, dt, offset, T):
    """Bit for bit what the same bytes at an aligned place give."""
    layer = Layer(gpu, oracle, dt, 4, 72, 512, 60)
    section = gpu.WeightsSection(np.concatenate([np.full(offset, 0xFF, np.uint8), layer.raw.reshape(-1)]))
    view = View(section, offset, dt, 4, 72, 512, layer.raw.size)
    x, ids = acts_for(61, T, 512), choices(62, T, 2, 4)
    want, got = (run_swiglu(gpu, rt, w, w, x, ids) for w in (layer, view))
    np.testing.assert_array_equal(bits(got), bits(want))
    h, weights = acts_for(63, T * 2, 512), np.random.default_rng(64).random((T, 2), np.float32)
    want, got = (run_combine(gpu, rt, w, h, weights, ids) for w in (layer, view))
    np.testing.assert_array_equal(bits(got), bits(want))


@pytest.mark.parametrize("dt,n", [(Q4_K, 4096), (Q6_K, 2816), (Q8_0, 2176)])
def test_experts_of_more_than_4_gib(gpu, rt, oracle, dt, n):
    """The same eight experts 64 times, those behind 4 GiB chosen."""
    small = Layer(gpu, oracle, dt, 8, n, 4096, 65)
    section = gpu.WeightsSection(np.tile(small.raw.reshape(-1), 64))
    big = View(section, 0, dt, 512, n, 4096, small.raw.size * 64)
    assert small.raw.size * 60 > 1 << 32
    for T in (2, 40, 600):
        x, ids = acts_for(66, T, 4096), np.random.default_rng(67).integers(480, 512, (T, 2)).astype(np.int32)
        want = run_swiglu(gpu, rt, small, small, x, ids % 8)
        np.testing.assert_array_equal(bits(run_swiglu(gpu, rt, big, big, x, ids)), bits(want))
        h, weights = acts_for(68, T * 2, 4096), np.random.default_rng(69).random((T, 2), np.float32)
        want = run_combine(gpu, rt, small, h, weights, ids % 8)
        np.testing.assert_array_equal(bits(run_combine(gpu, rt, big, h, weights, ids)), bits(want))
    big.w = None
    section.free()


def test_product_refusals(gpu, rt, oracle):
    """What the host turns away: nothing is launched."""
    L = gpu.load()
    gate, up = Layer(gpu, oracle, Q4_K, 4, 64, 256, 40), Layer(gpu, oracle, Q4_K, 4, 64, 256, 41)
    six, wide, b32 = (Layer(gpu, oracle, dt, 4, 64, k, 42) for dt, k in ((Q6_K, 256), (Q4_K, 512), (Q8_0, 256)))
    B = rt.DeviceBuffer
    x, h, w, plan, ws = B(1 << 16), B(1 << 16), B(1 << 12), B(1 << 12), B(1 << 20)
    nb = gpu.experts_plan_bytes(6, 2, 4)

    def swiglu(g=gate, u=up, n=4, T=6, top=2, x=x.ptr, h=h.ptr, plan=plan.ptr, nb=nb, ws=ws.ptr, wsb=1 << 20):
        return L.mimg_experts_swiglu_a8_dev(g.w.handle, u.w.handle, n, x, T, top, plan, nb, h, ws, wsb, None)

    def combine(d=gate, n=4, T=6, top=2, x=x.ptr, wt=w.ptr, h=h.ptr, plan=plan.ptr, nb=nb, ws=ws.ptr, wsb=1 << 20):
        return L.mimg_experts_combine_a8_dev(d.w.handle, n, x, wt, T, top, plan, nb, h, ws, wsb, None)

    for call in (swiglu, combine):
        for kw in (dict(n=3), dict(x=None), dict(h=None), dict(plan=None), dict(ws=None), dict(x=x.ptr + 8), dict(h=h.ptr + 4),
                   dict(ws=ws.ptr + 64), dict(plan=plan.ptr + 2), dict(h=x.ptr + 1024)):
            assert call(**kw) == -1, (call.__name__, kw)
        assert call(nb=nb - 4) == -6 and call(wsb=gpu.a8_workspace_bytes(6, 256) - 1) == -6
        assert call(T=0, x=None, h=None, plan=None, ws=None) == 0
    assert combine(wt=None) == -1 and combine(wt=h.ptr) == -1
    assert swiglu(u=wide) == -1
    assert swiglu(u=six) == 1 and swiglu(g=b32) == 1  # not handled: two dtypes
    assert L.mimg_experts_swiglu_a8_dev(gate.w.handle, 1 << 40, 4, x.ptr, 6, 2, plan.ptr, nb, h.ptr, ws.ptr, 1 << 20, None) == -4


def test_most_pairs(gpu, rt, oracle):
    """2^24 pairs of 1024 values (a launch of as many workgroups, 64 GiB): the
    same 2^18 over and over, each result as the one of these alone."""
    T, top, k, some = 1 << 20, 16, 1024, 1 << 14
    down = Layer(gpu, oracle, Q4_K, 16, 4, k, 50)
    ids = np.tile(choices(51, 64, top, 16), (some // 64, 1))
    weights = np.random.default_rng(52).random((some, top), np.float32)
    h = np.random.default_rng(53).standard_normal((some * top, k), np.float32)
    want = run_combine(gpu, rt, down, h, weights, ids)
    s, nb, wsb = rt.Stream(), gpu.experts_plan_bytes(T, top, 16), gpu.experts_combine_workspace_bytes(T, top, 4, k)
    dh, dw, di = rt.DeviceBuffer(T * top * k * 4), rt.DeviceBuffer(T * top * 4), rt.DeviceBuffer(T * top * 4)
    for b, a in ((dh, h), (dw, weights), (di, ids)):
        b.upload(a)
        at = a.nbytes
        while at < b.nbytes:
            rt.copy_async(b.ptr + at, b.ptr, at, s)
            at *= 2
    s.sync()
    plan, ws, y = rt.DeviceBuffer(nb), rt.DeviceBuffer(wsb), rt.DeviceBuffer(T * 16)
    gpu.experts_plan_dev(di.ptr, T, top, 16, plan.ptr, nb, s.handle)
    gpu.experts_combine_a8_dev(down.w, 16, dh.ptr, dw.ptr, T, top, plan.ptr, nb, y.ptr, ws.ptr, wsb, s.handle)
    s.sync()
    got = y.download(np.float32).reshape(T // some, some, 4)
    assert (bits(got) == bits(want)[None]).all()


@pytest.mark.parametrize("dt", [Q4_K, Q6_K, Q8_0])
@pytest.mark.parametrize("T", [2, 40, 300])
def test_products_of_scales_below_the_normal_ones(gpu, rt, oracle, dt, T):
    """x of 2^-118 and less: products of two scales that are subnormal float32;
    bit for bit what a token alone gives, for the K-quants what the oracle
    gives."""
    down = Layer(gpu, oracle, dt, 2, 64, 512, 70)
    h, ids = acts_for(71, T, 512), choices(72, T, 1, 2)
    h *= np.float32(2.0) ** -(118 + 3 * (np.arange(T)[:, None] % 7)).astype(np.float32)
    one = np.ones((T, 1), np.float32)
    got = run_combine(gpu, rt, down, h, one, ids)
    assert (got != 0).any()
    if dt != Q8_0:
        np.testing.assert_array_equal(bits(got), bits(expert_products(oracle, down, h, ids, True)[0]))
    alone = [run_combine(gpu, rt, down, h[t:t + 1], one[:1], ids[t:t + 1]) for t in range(0, T, 7)]
    np.testing.assert_array_equal(bits(got[::7]), bits(np.concatenate(alone)))
