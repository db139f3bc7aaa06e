"""Log probabilities, entropy and the largest alternatives (logprobs.hip)
against the 64-bit restatement. A log probability is (x - m) - log S: x - m and
its use in exponents to 2^-24 of it, sums over at most 32 values a thread and a
tree, so 2^-24 (2 |x - m| + |log S| + 128) bounds it; the entropy log S + T/S
2^-24 (128 + 128 T/S + |log S|). Ids are exact."""
import numpy as np
import pytest

import q8_ref

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def rt(gpu):
    import hiprt

    return hiprt


class Call:
    def __init__(self, gpu, rt, x, n, targets, top):
        self.gpu, self.rows, self.n, self.top = gpu, x.shape[0], n, top
        self.x = rt.DeviceBuffer.from_array(x)
        self.t = rt.DeviceBuffer.from_array(np.asarray(targets, np.int32))
        seven = lambda *s: rt.DeviceBuffer.from_array(np.full(s, 7, np.float32))  # noqa: E731
        self.lp, self.ent, self.ids, self.tlp = seven(self.rows + 8), seven(self.rows + 8), seven(self.rows * top + 8), seven(self.rows * top + 8)
        self.wsb = gpu.logprobs_workspace_bytes(self.rows, n, top)
        self.ws = seven(self.wsb // 4 + 8)
        self.ld = x.shape[1]

    def enqueue(self, s, off=0):
        """off: floats from the buffer's start to the logits."""
        p = lambda b: b.ptr if self.top else None  # noqa: E731
        self.gpu.logprobs_dev(self.x.ptr + 4 * off, self.rows, self.n, self.ld, self.t.ptr, self.top, self.lp.ptr, self.ent.ptr,
                              p(self.ids), p(self.tlp), self.ws.ptr, self.wsb, s.handle)

    def result(self):
        k = self.rows * self.top
        lp, ent, ids, tlp = (b.download(np.float32) for b in (self.lp, self.ent, self.ids, self.tlp))
        for b, m in ((lp, self.rows), (ent, self.rows), (ids, k), (tlp, k), (self.ws.download(np.float32), self.wsb // 4)):
            assert (b[m:] == 7).all()  # nothing past the end
        return lp[:self.rows], ent[:self.rows], ids[:k].view(np.int32).reshape(self.rows, -1), tlp[:k].reshape(self.rows, -1)


def run(gpu, rt, x, targets, top, n=None, off=0):
    c, s = Call(gpu, rt, x, n or x.shape[1], targets, top), rt.Stream()
    c.enqueue(s, off)
    s.sync()
    return c.result()


def check(got, x, targets, top):
    lp, ent, ids, tlp = q8_ref.logprobs(x, targets, top)
    x = x.astype(np.float64)
    m = x.max(-1)
    with np.errstate(invalid="ignore", divide="ignore"):
        log_s = np.log(np.exp(x - m[:, None]).sum(-1))
        given = np.where(lp == 0, 0, lp + log_s)
        tol = EPS * (2 * np.abs(given) + np.abs(log_s) + 128)
        assert (np.isneginf(got[0]) == np.isneginf(lp)).all()
        fin = np.isfinite(lp)
        assert (np.abs(got[0] - lp)[fin] <= tol[fin]).all(), np.abs(got[0] - lp)[fin].max()
        assert (np.abs(got[1] - ent) <= EPS * (128 + 128 * np.abs(ent - log_s) + np.abs(log_s))).all(), np.abs(got[1] - ent).max()
        assert np.array_equal(got[2], ids), np.argwhere(got[2] != ids)[:5]
        fin = np.isfinite(tlp)
        assert (np.isneginf(got[3]) == ~fin).all()
        assert (np.abs(got[3] - tlp)[fin] <= (EPS * (2 * np.abs(tlp) + 3 * np.abs(log_s)[:, None] + 128))[fin]).all()


@pytest.mark.parametrize("rows,n,top", [(1, 1, 1), (1, 3, 3), (2, 64, 64), (3, 100, 7), (5, 1023, 64), (2, 1024, 20), (4, 8191, 5),
                                        (1, 8192, 64), (3, 8193, 64), (2, 32003, 8), (1, 128256, 20), (9, 128256, 0), (40, 20000, 33),
                                        (2, 151936, 64), (1, 1 << 21, 64), (1, 600000, 1), (300, 77, 2), (70000, 5, 5)])
def test_rows(gpu, rt, rows, n, top):
    rng = np.random.default_rng(n + top)
    x = (rng.standard_normal((rows, n)) * rng.choice([0.1, 2.5, 30.0], (rows, 1))).astype(np.float32)
    t = rng.integers(0, n, rows)
    if rows > 2:
        t[0], t[1] = -1, n
    check(run(gpu, rt, x, t, top), x, t, top)


@pytest.mark.parametrize("n,ld,off", [(1000, 1001, 1), (8195, 9000, 3), (500, 500, 2), (33000, 33003, 1)])
def test_strides_and_alignment(gpu, rt, n, ld, off):
    """Rows apart by ld, at any 4-byte address; what lies behind a row is not
    part of it."""
    rows = 4
    rng = np.random.default_rng(n)
    flat = np.full(rows * ld + off + 4, np.nan, np.float32)
    x = rng.standard_normal((rows, n)).astype(np.float32)
    for r in range(rows):
        flat[off + r * ld:off + r * ld + n] = x[r]
    t = rng.integers(0, n, rows)
    c, s = Call(gpu, rt, flat[:rows * ld].reshape(rows, ld), n, t, 10), rt.Stream()
    c.x = rt.DeviceBuffer.from_array(flat)
    c.enqueue(s, off)
    s.sync()
    check(c.result(), x, t, 10)


@pytest.mark.parametrize("n", [300, 8192, 20000, 128256])
@pytest.mark.parametrize("top", [1, 8, 64])
def test_ties_masks_and_orders(gpu, rt, n, top):
    """Equal logits in every amount (ties to the lowest index), masked rows
    with fewer allowed tokens than alternatives, rising and falling rows, one
    token far above, zeros of both signs, the type's lowest value as a mask."""
    rng = np.random.default_rng(n + top)
    x = np.full((12, n), -np.inf, np.float32)
    x[0] = 1.5
    x[1] = rng.integers(0, 3, n)
    x[2, rng.choice(n, 5, replace=False)] = rng.standard_normal(5)
    x[3, n - 1] = 2
    x[4] = np.arange(n) * 1e-3
    x[5] = -np.arange(n) * 1e-3
    x[6] = rng.standard_normal(n)
    x[6, n // 2] = 60
    x[7] = np.where(np.arange(n) % 2, 0.0, -0.0)
    x[8] = np.finfo(np.float32).min
    x[8, [n // 3, n // 4]] = 1.0
    x[9, n // 2:] = 0.25
    x[10] = rng.integers(-1, 1, n)
    x[10, 200:260] = 3
    x[11] = -1e30
    t = rng.integers(0, n, 12)
    t[2], t[3], t[8], t[9] = int(np.argmax(x[2])), n - 1, n // 3, n - 1
    check(run(gpu, rt, x, t, top), x, t, top)


@pytest.mark.parametrize("top", [1, 5, 40, 64])
def test_few_equal_values_far_apart(gpu, rt, top):
    """Rows of a few values, each a handful of times all over a row: the ones
    that share the last place are the lowest indices, wherever they lie."""
    rng = np.random.default_rng(top)
    n = 20011
    x = np.full((24, n), -3.0, np.float32)
    for r in range(24):
        for value in (2.0, 1.0, 0.0, -1.0):
            many = int(rng.integers(0, [2, 9, 40, 90][r % 4]))
            x[r, rng.integers(0, n, many)] = value
        if r % 3 == 0:
            x[r, x[r] == -3.0] = -np.inf
            x[r, rng.integers(0, n)] = 0.5
    t = rng.integers(0, n, 24)
    t[::3] = [int(np.flatnonzero(x[r] == 0.5)[0]) for r in range(0, 24, 3)]
    check(run(gpu, rt, x, t, top), x, t, top)


def test_not_finite(gpu, rt):
    """NaN and +inf, and -inf alone, make a row's results NaN, no other row's;
    NaN is never among the alternatives."""
    n = 9000
    rng = np.random.default_rng(3)
    x = rng.standard_normal((5, n)).astype(np.float32)
    x[0, 17], x[1, 8999], x[2], x[3] = np.nan, np.inf, -np.inf, np.nan
    x[3, 40], x[3, 8500] = 1.0, 2.0
    lp, ent, ids, tlp = run(gpu, rt, x, np.zeros(5), 4)
    assert np.isnan(lp[:4]).all() and np.isnan(ent[:4]).all() and np.isnan(tlp[:4]).all() and np.isfinite(lp[4])
    clean = np.where(np.isnan(x), -np.inf, x)
    want = np.argsort(-clean, -1, kind="stable")[:, :4]
    assert np.array_equal(ids[[0, 1, 2, 4]], want[[0, 1, 2, 4]])
    assert list(ids[3]) == [8500, 40, -1, -1]


def test_outputs_may_be_left_out(gpu, rt):
    n, rows, top = 5000, 3, 6
    rng = np.random.default_rng(9)
    x = rng.standard_normal((rows, n)).astype(np.float32)
    full = run(gpu, rt, x, [5, 6, 7], top)
    c, s = Call(gpu, rt, x, n, [5, 6, 7], top), rt.Stream()
    for keep in range(4):
        outs = [b.ptr if i == keep else None for i, b in enumerate((c.lp, c.ent, c.ids, c.tlp))]
        gpu.logprobs_dev(c.x.ptr, rows, n, n, c.t.ptr if keep == 0 else None, top, *outs, c.ws.ptr, c.wsb, s.handle)
        s.sync()
    for a, b in zip(c.result(), full):
        assert np.array_equal(a, b)


def test_graph_replays(gpu, rt):
    rng = np.random.default_rng(2)
    xs = [rng.standard_normal((4, 40000)).astype(np.float32) for _ in range(3)]
    c, s = Call(gpu, rt, xs[0], 40000, [1, 2, 3, 4], 12), rt.Stream()
    g = rt.Graph(s, lambda: c.enqueue(s))
    for i in range(6):
        c.x.upload(xs[i % 3])
        rt.device_sync()
        g.launch(s)
        s.sync()
        check(c.result(), xs[i % 3], [1, 2, 3, 4], 12)
        c.enqueue(s)
        s.sync()
