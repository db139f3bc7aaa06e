"""Experts of so many rows that a launch of one workgroup for every few of them
passes the sizes that a grid may have: the same rows over and over, each result
as that of a matrix of these rows alone."""
import numpy as np
import pytest

from test_gpu_experts import Q4_K, Q8_0, acts_for, bits, run_combine, run_swiglu, rt  # noqa: F401

pytestmark = pytest.mark.gpu


class Repeated:
    """`experts` experts of n rows each, all of them `period` rows over and over
    (written on the device); alone: one expert of these rows."""

    def __init__(self, gpu, rt, oracle, dt, experts, n, period, k, seed):
        self.dt, self.experts, self.n, self.k = dt, experts, n, k
        raw = oracle.synthetic_weight(dt, period, k, seed=seed, scale=1 / np.sqrt(k)).reshape(-1)
        assert n % period == 0
        whole, s, at = rt.DeviceBuffer(raw.size * (experts * n // period)), rt.Stream(), raw.size
        whole.upload(raw)
        while at < whole.nbytes:
            rt.copy_async(whole.ptr + at, whole.ptr, min(at, whole.nbytes - at), s)
            at *= 2
        s.sync()
        self.w = gpu.Weight((whole.ptr, whole.nbytes), dt, experts * n, k, device=True)
        whole.free()
        self.alone = type("Alone", (), dict(dt=dt, experts=1, n=period, k=k, w=gpu.Weight(raw, dt, period, k)))


def same_rows(got, want):
    """got [rows, n] is want [rows, period] over and over, bit for bit."""
    for g, w in zip(got, want):
        assert (bits(g).reshape(-1, w.size) == bits(w)[None]).all()


def test_the_sum_over_rows_past_a_grid(gpu, rt, oracle):  # noqa: F811
    """Odd rows, so that a thread of the sum has one: 65538 workgroups of 256."""
    down = Repeated(gpu, rt, oracle, Q8_0, 1, 255 * 65795, 255, 32, 1)
    assert down.n % 4 and down.n > 65536 * 256
    h, ids = acts_for(2, 5, 32), np.zeros((5, 1), np.int32)
    weights = np.random.default_rng(3).random((5, 1), np.float32)
    same_rows(run_combine(gpu, rt, down, h, weights, ids), run_combine(gpu, rt, down.alone, h, weights, ids))


def test_the_sum_of_tokens_past_a_grid(gpu, rt, oracle):  # noqa: F811
    """270 tokens of 65538 workgroups each, more than 2^32 threads together."""
    T, n = 270, 255 * 65795
    down = Repeated(gpu, rt, oracle, Q8_0, 1, n, 255, 32, 4)
    h, ids = acts_for(5, T, 32), np.zeros((T, 1), np.int32)
    weights = np.random.default_rng(6).random((T, 1), np.float32)
    same_rows(run_combine(gpu, rt, down, h, weights, ids), run_combine(gpu, rt, down.alone, h, weights, ids))


@pytest.mark.parametrize("dt,k,n,T", [(Q8_0, 32, 1020 * 65794, 1), (Q8_0, 32, 1020 * 16449, 4), (Q4_K, 256, 1020 * 65794, 1),
                                       (Q4_K, 256, 1020 * 12337, 6)])
def test_few_pairs_of_rows_past_a_grid(gpu, rt, oracle, dt, k, n, T):  # noqa: F811
    """2^24 workgroups of 256 and more, where a pair runs its expert by itself."""
    assert n // 4 * T >= 1 << 24
    w = Repeated(gpu, rt, oracle, dt, 1, n, 1020, k, 7)
    x, ids = acts_for(8, T, k), np.zeros((T, 1), np.int32)
    same_rows(run_swiglu(gpu, rt, w, w, x, ids), run_swiglu(gpu, rt, w.alone, w.alone, x, ids))
    weights = np.random.default_rng(9).random((T, 1), np.float32)
    same_rows(run_combine(gpu, rt, w, x, weights, ids), run_combine(gpu, rt, w.alone, x, weights, ids))


def test_tiles_past_a_grid(gpu, rt, oracle):  # noqa: F811
    """A pair for each of 512 experts of 2^21 rows and more: more than 2^24 tiles
    of 64 rows, 36 GB of weights."""
    n = 96 * ((1 << 21) // 96 + 3)
    w = Repeated(gpu, rt, oracle, Q8_0, 512, n, 96, 32, 10)
    assert n * 512 > 64 << 24
    x = np.tile(acts_for(11, 16, 32), (32, 1))
    ids = np.random.default_rng(12).permutation(512).astype(np.int32)[:, None]
    alone = np.zeros((16, 1), np.int32)
    want = run_swiglu(gpu, rt, w.alone, w.alone, x[:16], alone)
    same_rows(run_swiglu(gpu, rt, w, w, x, ids), np.tile(want, (32, 1)))
    weights = np.tile(np.random.default_rng(13).random((16, 1), np.float32), (32, 1))
    want = run_combine(gpu, rt, w.alone, x[:16], weights[:16], alone)
    same_rows(run_combine(gpu, rt, w, x, weights, ids), np.tile(want, (32, 1)))


def test_experts_of_too_many_rows_are_not_handled(gpu, rt, oracle):  # noqa: F811
    """2^30 rows are an expert's most; nothing is launched."""
    n = (1 << 30) + 128
    w = Repeated(gpu, rt, oracle, Q8_0, 1, n, 128, 32, 14)
    L, B = gpu.load(), rt.DeviceBuffer
    x, weights, y, plan, ws = B(128), B(4), B(n * 4), B(1 << 12), B(n * 4 + (1 << 16))
    nb = gpu.experts_plan_bytes(1, 1, 1)
    assert L.mimg_experts_swiglu_a8_dev(w.w.handle, w.w.handle, 1, x.ptr, 1, 1, plan.ptr, nb, y.ptr, ws.ptr, ws.nbytes, None) == 1
    assert L.mimg_experts_combine_a8_dev(w.w.handle, 1, x.ptr, weights.ptr, 1, 1, plan.ptr, nb, y.ptr, ws.ptr, ws.nbytes, None) == 1
